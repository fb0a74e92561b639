// Attention of single tokens over the paged cache.
//
// Two sequences of 90,000 and 131,000 keys (8 key heads of 128, pages of 16): 165 us, 6.0 TB/s, 94 % of the
// rate of a copy; 32 sequences of 100 to 9,000 keys (8 heads of 64): 37 us, 4.3 TB/s, start and join included.
//
// Row (b, h) sees the keys [max(0, len_b - window), len_b) of its pages.  A
// decode step reads every key and value once for the G query heads that share
// it, about G flops a byte: HBM bound, so the kernel is built around keeping
// loads in flight and every SM busy whatever the lengths are.
//
//   * The work is one list of key tiles (128 keys of width 64, 64 of width 128: 32 KB) over (sequence, key head, tile of
//     16 query heads); CTA c of N takes an equal contiguous range of it.  A
//     range that cuts an item leaves a share (m, l, o) of it in the workspace, at
//     most two per CTA, and a second kernel joins the shares.  The split needs
//     only the lengths, which stay on the device: no host sync, and a captured step serves growing
//     lengths.
//   * Per CTA one TMA warp walks the page table (ids prefetched 32 at a time) and fills a ring of
//     tiles; four warps take a quarter of its keys each (mma.sync m16n8k16: a row
//     tile is 16 heads, far too few to feed tcgen05's 128 rows, and the tensor rate
//     is not the bound).  Each warp keeps its own running
//     maximum, sum and 16 x D output; the four are joined once per item.
//   * Rows of a group share their first keys (the prefix): the tensor-core kernel of attn_tc.cu reads
//     those once for all rows of the group, this one takes the keys behind them, and the join
//     adds the prefix's shares.  This kernel may start beside the prefix kernel (programmatic launch), but not
//     on the same SMs (195 and 105 KB of shared memory): with a prefix item on every SM it runs as those
//     finish.  The join waits for both.
#include <algorithm>

#include "attn_common.cuh"
#include "attn_kernels.cuh"
#include "tc_common.cuh"

namespace klc {
namespace attn {

using namespace tc;

namespace {

constexpr int kThreads = 160;  // four math warps, one TMA warp
constexpr int kCtasPerSm = 2;
constexpr int kRowTile = 16;
// What starting and ending an item costs a CTA, in tiles (queries, joining the warps, the output): counted into the split, or
// CTAs that get many short sequences finish last (32 sequences of 100 to 9000 keys: 60 / 51 / 46 / 44 / 43 us with 0 / 1 / 2 / 3 / 4).
constexpr int kItemCost = 3;

// A sequence in a CTA's plan: units (tiles, and kItemCost per item) of the sequences before it over one key head and row tile, and the keys [klo, len) its own pages contribute.
struct Seq {
  int cum, klo, len, prefix;
};

template <int D>
struct DCfg {
  static constexpr int kTileKeys = D == 64 ? 128 : 64;        // 32 KB of keys and values either way
  static constexpr int kGroups = kTileKeys / 64;              // groups of 16 keys a warp takes of a tile
  static constexpr int kChunks = D / 64;
  static constexpr int kHalf = kTileKeys * D * 2;             // bytes of a key (or value) tile
  static constexpr int kStage = 2 * kHalf;                    // keys and values
  static constexpr int kStages = 3;                           // 96 KB in flight per CTA
  static constexpr int kOld = D + 8;                          // row pitch of the join buffer (floats)
  static constexpr int OFF_RING = 0;
  static constexpr int OFF_O = kStages * kStage;              // [16][kOld] fp32
  static constexpr int OFF_ML = OFF_O + kRowTile * kOld * 4;  // [4][16] (m, l)
  static constexpr int OFF_BAR = OFF_ML + 4 * kRowTile * 8;
  static constexpr int OFF_MISC = OFF_BAR + 2 * kStages * 8;
  static constexpr int OFF_SEQ = OFF_MISC + 64;               // [batch + 1] Seq
  static size_t smem(int64_t batch) { return size_t(OFF_SEQ) + size_t(batch + 1) * sizeof(Seq) + 1024; }
};

__device__ __forceinline__ int prefix_of(const DecodeParams& p, int b) {
  if (p.groups == 0) return 0;
  int lo = 0, hi = p.groups;  // last group whose start is <= b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.group_starts[mid] <= b) lo = mid;
    else hi = mid;
  }
  if (b < p.group_starts[lo] || b >= p.group_starts[lo + 1]) return 0;
  const int pre = p.prefix_lens[lo];
  return pre < 0 || pre % p.page_size != 0 || pre > p.table_width * p.page_size ? 0 : pre;  // reported by the prefix kernel
}

__device__ __forceinline__ Seq seq_of(const DecodeParams& p, int b, bool report) {
  int len = p.lens[b];
  if (len < 0 || int64_t(len) > int64_t(p.table_width) * p.page_size) {
    if (report) record_fault(p.status, KLC_ERR_DEVICE_FAULT, 510, b);
    len = 0;
  }
  Seq s;
  s.cum = 0;
  s.prefix = prefix_of(p, b);
  s.klo = max(p.window > 0 ? max(0, len - p.window) : 0, s.prefix);
  s.len = len;
  return s;
}
template <int TK>
__device__ __forceinline__ int units_of(const Seq& s) {
  return s.len > s.klo ? (s.len + TK - 1) / TK - s.klo / TK + kItemCost : 0;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Elem<T>::kMmaFormat == 1)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// barrier of the four math warps, with and without the conjunction of their flags
__device__ __forceinline__ void math_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool math_sync_and(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(uint32_t(ok))
      : "memory");
  return all != 0;
}

// A run of one item's units in a CTA's range: kItemCost units, then its tiles.  A run that ends inside the former has no
// tile (the next CTA takes the item).
struct Run {
  int b, hr;          // sequence; key head * row tiles + row tile
  int units;          // of the run
  int tile, n;        // first tile (counted from the item's first) and number of tiles
  int tiles;          // of the whole item
};

__device__ __forceinline__ Run run_at(const Seq* seqs, int batch, int hrs, int64_t x, int64_t end) {
  int lo = 0, hi = batch;  // last sequence with cum * hrs <= x (its count is positive, since x is inside)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (int64_t(seqs[mid].cum) * hrs <= x) lo = mid;
    else hi = mid;
  }
  Run r;
  r.b = lo;
  const int cum = seqs[lo].cum, units = seqs[lo + 1].cum - cum;
  const uint32_t rel = uint32_t(x - int64_t(cum) * hrs);  // units * hrs of one sequence: fits (checked by the host)
  r.hr = int(rel / uint32_t(units));
  const int u0 = int(rel - uint32_t(r.hr) * uint32_t(units));
  r.units = int(min(int64_t(units - u0), end - x));
  r.tiles = units - kItemCost;
  r.tile = max(0, u0 - kItemCost);
  r.n = max(0, u0 + r.units - kItemCost) - r.tile;
  return r;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
attn_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const DecodeParams p) {
  using C = DCfg<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int TK = C::kTileKeys;
  Seq* seqs = reinterpret_cast<Seq*>(smem + C::OFF_SEQ);
  int* scan_s = reinterpret_cast<int*>(smem + C::OFF_MISC + 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC);
  const Ctl ctl{abort_flag, p.status};
  const uint32_t bar0 = smem_u32(smem + C::OFF_BAR);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };

  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32 * 4) {
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  pdl_trigger();
  if (!p.after_prefix) pdl_wait();  // started by the prefix kernel, which has waited for what came before

  // ---- prefix sums of the sequences' tiles
  const int per = (p.batch + kThreads - 1) / kThreads, b0 = min(p.batch, tid * per), b1 = min(p.batch, b0 + per);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    seqs[b] = seq_of(p, b, blockIdx.x == 0);
    mine += units_of<TK>(seqs[b]);
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan_s[warp] = incl;
  __syncthreads();
  int at = incl - mine;
  for (int w = 0; w < warp; ++w) at += scan_s[w];
  for (int b = b0; b < b1; ++b) {
    seqs[b].cum = at;
    if (blockIdx.x == 0) p.cum[b] = at;
    at += units_of<TK>(seqs[b]);
    if (b == p.batch - 1) {
      seqs[p.batch].cum = at;
      if (blockIdx.x == 0) p.cum[p.batch] = at;
    }
  }
  __syncthreads();
  const int hrs = p.kv_heads * p.row_tiles;
  const int64_t total = int64_t(seqs[p.batch].cum) * hrs;
  const int64_t nc = min(int64_t(gridDim.x), total);  // CTAs with a unit at least
  const int64_t x0 = blockIdx.x < nc ? total * blockIdx.x / nc : 0, x1 = blockIdx.x < nc ? total * (blockIdx.x + 1) / nc : 0;

  if (warp == 4) {
    // ---------------------------------------------------------------- loads
    const int box = min(p.page_size, TK), parts = TK / box;
    const int boxes = parts * C::kChunks * 2;  // at most 16: lane j issues box j
    const int bkv = lane / (parts * C::kChunks), bc = (lane / parts) % C::kChunks, bp = lane % parts;
    uint32_t issued = 0;
    bool ok = true;
    for (int64_t x = x0; x < x1 && ok;) {
      const Run r = run_at(seqs, p.batch, hrs, x, x1);
      const Seq sp = seqs[r.b];
      const int tile0 = sp.klo / TK;
      const int kvh = r.hr / p.row_tiles;
      const int32_t* table = p.block_table + int64_t(r.b) * p.table_stride;
      int have = -1, cached = 0;  // lane's page id of table entry have + lane
      for (int i = 0; i < r.n && ok; ++i, ++issued) {
        const int key0 = (tile0 + r.tile + i) * TK;
        const int e0 = key0 / p.page_size, e1 = (key0 + TK - 1) / p.page_size;
        if (have < 0 || e1 >= have + 32) {
          have = e0;
          const int e = have + lane;
          cached = int64_t(e) * p.page_size < sp.len && int64_t(e + 1) * p.page_size > sp.klo ? table[e] : -1;
        }
        const int key = key0 + bp * box;
        int page = __shfl_sync(0xffffffffu, cached, (key / p.page_size - have) & 31);
        if (key >= sp.len || key + box <= sp.klo) {
          page = int(p.pages);  // no key of the row in this box: zeros (a coordinate past the pool)
        } else if (page < 0 || page >= p.pages) {
          record_fault(p.status, KLC_ERR_DEVICE_FAULT, 511, page);
          page = int(p.pages);
        }
        const int s = issued % C::kStages;
        ok = wait_bar(empty(s), ((issued / C::kStages) & 1) ^ 1, ctl, 512);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        if (lane == 0) mbar_arrive_expect_tx(full(s), uint32_t(C::kStage));
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(smem_u32(smem + C::OFF_RING + s * C::kStage + bkv * C::kHalf + bc * (TK * 128) + bp * box * 128),
                      bkv ? &map_v : &map_k, bc * 64, key % p.page_size, kvh, page, full(s));
      }
      x += r.units;
    }
    if (!ok) drain_ring(full(0), C::kStages, issued);
  } else {
    // ---------------------------------------------------------------- math
    float* osum = reinterpret_cast<float*>(smem + C::OFF_O);
    float2* ml = reinterpret_cast<float2*>(smem + C::OFF_ML);
    const int G = p.group, row = lane >> 2, quad = lane & 3;
    uint32_t used = 0;
    bool ok = true;
    for (int64_t x = x0; x < x1 && ok;) {
      const Run r = run_at(seqs, p.batch, hrs, x, x1);
      const Seq sp = seqs[r.b];
      const int tile0 = sp.klo / TK;
      if (r.n == 0) break;  // the range ends inside the item's start
      const int kvh = r.hr / p.row_tiles, rt = r.hr - kvh * p.row_tiles;
      const int rows = min(kRowTile, G - rt * kRowTile);
      const int head0 = kvh * G + rt * kRowTile;
      const T* q = reinterpret_cast<const T*>(p.q) + int64_t(r.b) * p.q_ts + int64_t(head0) * p.q_hs;
      uint32_t qf[D / 16][4];
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int rr = row + (j & 1) * 8;
          qf[kk][j] = rr < rows ? *reinterpret_cast<const uint32_t*>(q + int64_t(rr) * p.q_hs + kk * 16 + quad * 2 + (j >> 1) * 8) : 0u;
        }
      float o[D / 8][4];
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

      for (int i = 0; i < r.n; ++i, ++used) {
        const int s = used % C::kStages;
        ok = wait_bar(full(s), (used / C::kStages) & 1, ctl, 513);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        const uint32_t kbase = smem_u32(smem + C::OFF_RING + s * C::kStage), vbase = kbase + C::kHalf;
        // S = Q K^T for this warp's kGroups x 16 keys
        constexpr int NG = C::kGroups;
        float sc[2 * NG][4] = {};
        const int wkey = warp * (16 * NG);  // the warp's first key in the tile
        const int krow = wkey + ((lane >> 4) << 3) + (lane & 7);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const int ch = (kk * 2 + ((lane >> 3) & 1)) & 7;
#pragma unroll
          for (int gk = 0; gk < NG; ++gk) {
            uint32_t kf[4];
            ldsm4(kbase + (kk >> 2) * (TK * 128) + (krow + 16 * gk) * 128 + ((ch ^ (krow & 7)) << 4), kf);
            mma16816<T>(sc[2 * gk], qf[kk], kf[0], kf[1]);
            mma16816<T>(sc[2 * gk + 1], qf[kk], kf[2], kf[3]);
          }
        }
        const int key = (tile0 + r.tile + i) * TK + wkey;
        uint32_t vmask[2 * NG];
#pragma unroll
        for (int h = 0; h < 2 * NG; ++h) vmask[h] = 0xffffffffu;
        if (key < sp.klo || key + 16 * NG > sp.len) {
          // hidden keys: no weight, and a value row of zeros (what is stored there may not be a number)
#pragma unroll
          for (int h = 0; h < 2 * NG; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int kx = key + h * 8 + quad * 2 + e;
              if (kx < sp.klo || kx >= sp.len) {
                sc[h][e] = sc[h][e + 2] = -INFINITY;
                vmask[h] &= e ? 0x0000ffffu : 0xffff0000u;
              }
            }
        }
        uint32_t pf[NG][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // rows `row` and `row + 8`
          float mx = sc[0][2 * h];
#pragma unroll
          for (int c = 0; c < 2 * NG; ++c) mx = max3_nan(mx, sc[c][2 * h], sc[c][2 * h + 1]);
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * p.scale_log2 - Elem<T>::kTopLog2;  // the largest numerator: 2^kTopLog2
          if (mx > m[h] || mx != mx) {  // a NaN stays: nothing is larger, and a tile without keys must not take its place
            const float f = exp2_approx(m[h] - mx);  // 0 from the initial -inf
            m[h] = mx;
            l[h] *= f;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              o[j][2 * h] *= f;
              o[j][2 * h + 1] *= f;
            }
          }
          const float ref = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
          for (int gk = 0; gk < NG; ++gk) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) e[c] = exp2_approx(fmaf(sc[2 * gk + (c >> 1)][2 * h + (c & 1)], p.scale_log2, -ref));
            l[h] += (e[0] + e[1]) + (e[2] + e[3]);  // this lane's keys; summed over the quad at the end
            pf[gk][h] = Elem<T>::pack(e[0], e[1]);
            pf[gk][2 + h] = Elem<T>::pack(e[2], e[3]);
          }
        }
        // O += P V
        const int vrow = wkey + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          const int ch = (j * 2 + (lane >> 4)) & 7;
#pragma unroll
          for (int gk = 0; gk < NG; ++gk) {
            uint32_t vf[4];
            ldsm4_t(vbase + (j >> 2) * (TK * 128) + (vrow + 16 * gk) * 128 + ((ch ^ (vrow & 7)) << 4), vf);
            mma16816<T>(o[2 * j], pf[gk], vf[0] & vmask[2 * gk], vf[1] & vmask[2 * gk + 1]);
            mma16816<T>(o[2 * j + 1], pf[gk], vf[2] & vmask[2 * gk], vf[3] & vmask[2 * gk + 1]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      }
      // ---- join the four warps: scale to the common maximum, add in warp order
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (quad == 0) ml[warp * kRowTile + row + 8 * h] = make_float2(m[h], l[h]);
      }
      // a warp whose wait gave up still comes here, and then all four leave together
      if (!(ok = math_sync_and(ok))) break;
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max_nan(top, ml[w * kRowTile + row + 8 * h].x);
        f[h] = m[h] == -INFINITY ? 0.f : exp2_approx(m[h] - top);
      }
      for (int w = 0; w < 4; ++w) {
        if (w == warp) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float2* dst = reinterpret_cast<float2*>(osum + (row + 8 * h) * C::kOld + j * 8 + quad * 2);
              float2 a = make_float2(o[j][2 * h] * f[h], o[j][2 * h + 1] * f[h]);
              if (w > 0) {
                const float2 c = *dst;
                a.x += c.x;
                a.y += c.y;
              }
              *dst = a;
            }
        }
        math_sync();
      }
      // ---- out: the finished row, or the CTA's share of a cut one
      const bool cut = r.n != r.tiles, whole = !cut && sp.prefix == 0;
      const int slot = 2 * blockIdx.x + (x > x0 ? 1 : 0);
      constexpr int kPerRow = D / 8;  // eight values a thread
      for (int idx = tid; idx < rows * kPerRow; idx += 128) {
        const int rr = idx / kPerRow, c8 = idx - rr * kPerRow;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max_nan(top, ml[w * kRowTile + rr].x);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float2 a = ml[w * kRowTile + rr];
          if (a.x != -INFINITY) sum += a.y * exp2_approx(a.x - top);
        }
        const float* src = osum + rr * C::kOld + c8 * 8;
        if (whole) {
          const int head = head0 + rr;
          float inv, lse;
          finish_row(top, sum, p.sinks != nullptr, p.sinks != nullptr ? p.sinks[head] * kLog2e : 0.f, &inv, &lse);
          uint4 w;
          w.x = Elem<T>::pack(src[0] * inv, src[1] * inv);
          w.y = Elem<T>::pack(src[2] * inv, src[3] * inv);
          w.z = Elem<T>::pack(src[4] * inv, src[5] * inv);
          w.w = Elem<T>::pack(src[6] * inv, src[7] * inv);
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + int64_t(r.b) * p.out_ts + int64_t(head) * p.out_hs + c8 * 8) = w;
          if (p.lse != nullptr && c8 == 0) p.lse[int64_t(r.b) * p.heads + head] = lse;
        } else {
          // a CTA has at most two cut items; an uncut one behind a prefix goes next to the prefix's shares
          const int64_t own = (int64_t(p.splits) * p.batch + r.b) * p.heads + head0 + rr;
          float4* dst = reinterpret_cast<float4*>((cut ? p.part_o + (int64_t(slot) * kRowTile + rr) * D : p.prefix_o + own * D) + c8 * 8);
          dst[0] = *reinterpret_cast<const float4*>(src);
          dst[1] = *reinterpret_cast<const float4*>(src + 4);
          if (c8 == 0) *(cut ? p.part_ml + slot * kRowTile + rr : p.prefix_ml + own) = make_float2(top, sum);
        }
      }
      math_sync();  // the buffers are free for the next item
      x += r.units;
    }
  }
  if (p.after_prefix) pdl_wait();  // this grid ends after the prefix kernel: the join waits for both
}

// ---------------------------------------------------------------------------
// Join of the shares: one warp per (row, head).  The shares are read in a fixed
// order (prefix splits, then CTAs), so results do not depend on timing.
// ---------------------------------------------------------------------------
constexpr int kJoinWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const DecodeParams p, int ctas) {
  constexpr int V = D / 32;  // values a lane
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int64_t rid = int64_t(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
  if (rid >= int64_t(p.batch) * p.heads) return;
  const int b = int(rid / p.heads), head = int(rid - int64_t(b) * p.heads);
  const int kvh = head / p.group, g = head - kvh * p.group, rt = g / kRowTile, rr = g - rt * kRowTile;
  const int hrs = p.kv_heads * p.row_tiles;
  const int c0 = p.cum[b], units = p.cum[b + 1] - c0;
  const int64_t total = int64_t(p.cum[p.batch]) * hrs, nc = min(int64_t(ctas), total);
  const bool prefix = prefix_of(p, b) > 0;
  int first = 0, last = -1;  // CTAs that hold shares of the item
  int64_t i0 = 0;
  if (units > 0) {  // CTA of a unit u: the last one whose range starts at or before u
    i0 = int64_t(c0) * hrs + int64_t(kvh * p.row_tiles + rt) * units;
    first = int(((i0 + kItemCost + 1) * nc - 1) / total);
    last = int(((i0 + units) * nc - 1) / total);
  }
  if (!prefix && first == last) return;  // written by the decode kernel

  // Shares: the prefix's splits, then the row's own keys (one share if uncut, else one per CTA: the first CTA's second
  // slot if the item starts inside its range, the first slot of the others).  Lane i holds share i's (m, l).
  const int skip = prefix ? 0 : p.splits, own = last - first + 1, n = p.splits + own - skip;
  const int64_t pre_row = int64_t(b) * p.heads + head, pre_step = int64_t(p.batch) * p.heads;
  const bool inside = own > 1 && total * first / nc < i0;
  auto share = [&](int i) -> int64_t {  // row index into the prefix arrays, or ~(row index) into the CTAs' shares
    i += skip;
    if (i < p.splits || own == 1) return pre_row + i * pre_step;
    const int c = i - p.splits;
    return ~(int64_t(2 * (first + c) + (c == 0 && inside ? 1 : 0)) * kRowTile + rr);
  };
  float top = -INFINITY, sum = 0.f, acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  for (int i0s = 0; i0s < n; i0s += 32) {
    const int mine = i0s + lane;
    int64_t at = 0;
    float2 a = make_float2(-INFINITY, 0.f);
    if (mine < n) {
      at = share(mine);
      a = at >= 0 ? p.prefix_ml[at] : p.part_ml[~at];
    }
    const float was = top;
    float mx = a.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    top = fmaxf(top, mx);
    const float f = a.x == -INFINITY ? 0.f : exp2_approx(a.x - top);  // 0: no keys, and its output was not written
    float part = warp_sum(a.y * f);
    const float back = was == -INFINITY ? 0.f : exp2_approx(was - top);
    sum = sum * back + part;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] *= back;
    const int count = min(32, n - i0s);
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      const int64_t r = __shfl_sync(0xffffffffu, at, i);
      if (fi == 0.f) continue;
      const float* src = (r >= 0 ? p.prefix_o + r * D : p.part_o + ~r * D) + lane * V;
      if constexpr (V == 2) {
        const float2 x = *reinterpret_cast<const float2*>(src);
        acc[0] += x.x * fi;
        acc[1] += x.y * fi;
      } else {
        const float4 x = *reinterpret_cast<const float4*>(src);
        acc[0] += x.x * fi;
        acc[1] += x.y * fi;
        acc[2] += x.z * fi;
        acc[3] += x.w * fi;
      }
    }
  }
  float inv, lse;
  finish_row(top, sum, p.sinks != nullptr, p.sinks != nullptr ? p.sinks[head] * kLog2e : 0.f, &inv, &lse);
  uint32_t w[V / 2];
#pragma unroll
  for (int j = 0; j < V / 2; ++j) w[j] = Elem<T>::pack(acc[2 * j] * inv, acc[2 * j + 1] * inv);
  uint32_t* dst = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + int64_t(b) * p.out_ts + int64_t(head) * p.out_hs + lane * V);
#pragma unroll
  for (int j = 0; j < V / 2; ++j) dst[j] = w[j];
  if (p.lse != nullptr && lane == 0) p.lse[int64_t(b) * p.heads + head] = lse;
}

template <typename T, int D>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const DecodeParams& p, int ctas, cudaStream_t s) {
  const size_t smem = DCfg<D>::smem(p.batch);
  auto kernel = attn_decode_kernel<T, D>;
  static SmemLimit limit;
  int st = limit.raise(reinterpret_cast<const void*>(kernel), DCfg<D>::smem(kMaxBatch));
  if (st != KLC_OK) return st;
  KLC_CUDA(launch_chain(kernel, dim3(unsigned(ctas)), dim3(kThreads), smem, s, 0, mk, mv, p));
  KLC_LAUNCH_CHECK("attn_decode");
  const int64_t rows = int64_t(p.batch) * p.heads;
  KLC_CUDA(launch_chain(attn_join_kernel<T, D>, dim3(unsigned((rows + kJoinWarps - 1) / kJoinWarps)), dim3(kJoinWarps * 32), 0, s, 0,
                        p, ctas));
  KLC_LAUNCH_CHECK("attn_join");
  return KLC_OK;
}

struct Plan {
  int ctas, splits;
  size_t off_cum, off_ml, off_o, off_pml, off_po, bytes;
};

Plan plan_of(const klc_attn_dims& d, int64_t batch, int64_t groups) {
  Plan pl{};
  const int sms = sm_count(), G = d.heads / d.kv_heads;
  pl.ctas = sms * kCtasPerSm;
  if (groups > 0) {
    // row-tile pairs of the prefix kernel; enough key splits to give every SM one
    const int tok = 2 * (128 / G);
    const int64_t pairs = std::min(batch, groups == 1 ? (batch + tok - 1) / tok : batch / tok + groups);
    pl.splits = int(std::max<int64_t>(1, std::min<int64_t>(16, sms / std::max<int64_t>(1, pairs * d.kv_heads))));
  }
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t a = off;
    off = align_up(off + n, 256);
    return a;
  };
  pl.off_cum = take(size_t(batch + 1) * 4);
  pl.off_ml = take(size_t(pl.ctas) * 2 * kRowTile * 8);
  pl.off_o = take(size_t(pl.ctas) * 2 * kRowTile * d.head_dim * 4);
  const size_t rows = (pl.splits > 0 ? size_t(pl.splits) + 1 : 0) * size_t(batch) * size_t(d.heads);
  pl.off_pml = take(rows * 8);
  pl.off_po = take(rows * size_t(d.head_dim) * 4);
  pl.bytes = off;
  return pl;
}

int check_decode_dims(const klc_attn_dims* dims, int64_t batch, int64_t groups) {
  const char* who = "klc_attn_decode";
  KLC_CHECK_ARG(dims != nullptr, "klc_attn_decode: null dims");
  int st = check_heads(who, dims->dtype, dims->heads, dims->kv_heads, dims->head_dim);
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(batch >= 0 && groups >= 0, "klc_attn_decode: negative size");
  if (batch > kMaxBatch) return fail(KLC_ERR_UNSUPPORTED, "klc_attn_decode: at most 4096 sequences");
  KLC_CHECK_ARG(groups <= batch, "klc_attn_decode: more groups than sequences");
  return KLC_OK;
}

}  // namespace
}  // namespace attn
}  // namespace klc

extern "C" int klc_attn_decode_workspace_size(const klc_attn_dims* dims, int64_t batch, int64_t groups, size_t* out_bytes) {
  using namespace klc;
  using namespace klc::attn;
  const int st = check_decode_dims(dims, batch, groups);
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(out_bytes != nullptr, "klc_attn_decode_workspace_size: null output");
  *out_bytes = plan_of(*dims, batch, groups).bytes;
  return KLC_OK;
}

extern "C" int klc_attn_decode(const klc_attn_dims* dims, const void* q, int64_t q_token_stride, int64_t q_head_stride,
                               const void* k_pages, const void* v_pages, int64_t pages, int page_size, int64_t page_stride,
                               const int32_t* block_table, int64_t table_width, int64_t table_stride, const int32_t* lens,
                               int64_t batch, const int32_t* group_starts, const int32_t* prefix_lens, int64_t groups,
                               const float* sinks, void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse,
                               void* workspace, size_t workspace_bytes, void* status, void* stream) {
  using namespace klc;
  using namespace klc::attn;
  int st = check_decode_dims(dims, batch, groups);
  if (st == KLC_OK) st = check_scale("klc_attn_decode", dims->scale);
  if (st != KLC_OK) return st;
  KLC_CHECK_ARG(dims->window >= 0, "klc_attn_decode: negative window");
  KLC_CHECK_ARG(page_size_ok(page_size), "klc_attn_decode: page_size must be 16, 32, 64 or 128");
  KLC_CHECK_ARG(pages >= 1 && pages < (1 << 30), "klc_attn_decode: pages must be between 1 and 2^30");
  KLC_CHECK_ARG(table_width >= 0 && table_width < (int64_t(1) << 31) && table_stride >= table_width, "klc_attn_decode: bad block table width or stride");
  KLC_CHECK_ARG(table_width * page_size < (int64_t(1) << 31) && batch * (table_width * page_size / 64 + 1 + kItemCost) < (int64_t(1) << 31) &&
                    int64_t(dims->heads) * (table_width * page_size / 64 + 1 + kItemCost) < (int64_t(1) << 31),
                "klc_attn_decode: the block table covers too many keys");
  if (batch == 0) return KLC_OK;
  const int d = dims->head_dim;
  KLC_CHECK_ARG(k_pages != nullptr && v_pages != nullptr && lens != nullptr, "klc_attn_decode: null pointer");
  KLC_CHECK_ARG(block_table != nullptr || table_width == 0, "klc_attn_decode: null block table");
  KLC_CHECK_ARG(groups == 0 || (group_starts != nullptr && prefix_lens != nullptr), "klc_attn_decode: null groups");
  KLC_CHECK_ARG(aligned16(k_pages) && aligned16(v_pages), "klc_attn_decode: the pools must be 16-byte aligned");
  KLC_CHECK_ARG(page_stride % 8 == 0 && page_stride >= int64_t(dims->kv_heads) * page_size * d && page_stride < (int64_t(1) << 38),
                "klc_attn_decode: page_stride must be a multiple of 8 and hold a page");
  if ((st = check_rows("klc_attn_decode", "q", q, batch, q_token_stride, q_head_stride, dims->heads, d)) != KLC_OK) return st;
  if ((st = check_rows("klc_attn_decode", "out", out, batch, out_token_stride, out_head_stride, dims->heads, d)) != KLC_OK) return st;
  const Plan pl = plan_of(*dims, batch, groups);
  KLC_CHECK_ARG(workspace != nullptr && aligned16(workspace), "klc_attn_decode: the workspace must be 16-byte aligned");
  if (workspace_bytes < pl.bytes)
    return fail(KLC_ERR_WORKSPACE, "klc_attn_decode: workspace of " + std::to_string(workspace_bytes) + " bytes, need " +
                                       std::to_string(pl.bytes));
  unsigned char* ws = reinterpret_cast<unsigned char*>(workspace);
  const int G = dims->heads / dims->kv_heads;

  DecodeParams p{};
  p.q = q;
  p.q_ts = q_token_stride;
  p.q_hs = q_head_stride;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.table_width = int(table_width);
  p.pages = pages;
  p.page_size = page_size;
  p.lens = lens;
  p.batch = int(batch);
  p.group_starts = group_starts;
  p.prefix_lens = prefix_lens;
  p.groups = int(groups);
  p.heads = dims->heads;
  p.kv_heads = dims->kv_heads;
  p.group = G;
  p.row_tiles = (G + kRowTile - 1) / kRowTile;
  p.scale_log2 = dims->scale * kLog2e;
  p.window = dims->window;
  p.sinks = sinks;
  p.out = out;
  p.out_ts = out_token_stride;
  p.out_hs = out_head_stride;
  p.lse = lse;
  p.status = reinterpret_cast<DeviceStatus*>(status);
  p.cum = reinterpret_cast<int*>(ws + pl.off_cum);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.off_ml);
  p.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  p.prefix_ml = reinterpret_cast<float2*>(ws + pl.off_pml);
  p.prefix_o = reinterpret_cast<float*>(ws + pl.off_po);
  p.splits = pl.splits;

  cudaStream_t s = as_stream(stream);
  if (groups > 0) {
    if ((st = launch_prefix(*dims, p, q, k_pages, v_pages, page_stride, s)) != KLC_OK) return st;
    p.after_prefix = pdl_enabled();
  }
  CUtensorMap mk, mv;
  const int box = std::min(page_size, d == 64 ? DCfg<64>::kTileKeys : DCfg<128>::kTileKeys);
  if ((st = pool_map(&mk, dims->dtype, d, k_pages, pages, dims->kv_heads, page_size, page_stride, box)) != KLC_OK) return st;
  if ((st = pool_map(&mv, dims->dtype, d, v_pages, pages, dims->kv_heads, page_size, page_stride, box)) != KLC_OK) return st;
  if (dims->dtype == KLC_BF16)
    return d == 64 ? launch<__nv_bfloat16, 64>(mk, mv, p, pl.ctas, s) : launch<__nv_bfloat16, 128>(mk, mv, p, pl.ctas, s);
  return d == 64 ? launch<__half, 64>(mk, mv, p, pl.ctas, s) : launch<__half, 128>(mk, mv, p, pl.ctas, s);
}
