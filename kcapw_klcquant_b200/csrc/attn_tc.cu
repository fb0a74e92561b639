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
//   8, 10     MMA issuer of row tile 0 / 1 (one thread); settles values that not all rows of the item see
//   9         finds the items; TMA producer (queries, then a ring of key and value tiles)
// Per key tile and row tile: S = Q K^T into TMEM (128 fp32 columns), the
// softmax thread reads its row and writes P as 16-bit pairs, and O += P V
// reads P from TMEM.  The tensor pipe works on one row tile while the other is
// in its softmax.  Row statistics are fp32.  O is rescaled only when a row's
// maximum has grown by more than 2^8 (f16: 2^4) since the last rescale (a late rescale, like
// exponentials shared out between two pipes, is a published idea for this kind of kernel): until then
// P is at most 2^8 (f16: 2^15), inside the type's range, and its relative rounding
// (2^-8 / 2^-11, the price of a 16-bit P operand) does not depend on the reference.
// f16 keeps that for weights down to 2^-25 of the row's largest; 2^-36 is the smallest that counts.
//
// Bound: with D = 128 the chain softmax -> P V -> next S of a row tile (TMEM
// has no room for a second S), with D = 64 the latencies of two softmax warps a
// scheduler (no pipe is full).  16221
// tokens, 32 / 8 heads of 128: 2.02 ms, 1.07 PFLOP/s, 62 % of the burst rate of
// a library product (74 % of its sustained one); 6016 tokens, 64 / 8 heads of
// 64: 408 us, 727 TFLOP/s.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "attn_kernels.cuh"
#include "tc_common.cuh"

namespace klc {
namespace attn {

using namespace tc;

namespace {

// try_wait that lets the hardware hold the warp for up to `ns`, so that waiting warps leave the issue slots to the others
__device__ __forceinline__ bool mbar_try_wait_ns(uint32_t bar, uint32_t parity, uint32_t ns) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(ns)
      : "memory");
  return ok != 0;
}

// wait_bar with everything but the first try out of line (the waits are many, and code size costs here)
__device__ __noinline__ bool wait_bar_long(uint32_t bar, uint32_t parity, const Ctl& c, int site) {
  const long long t0 = clock64();
  while (!mbar_try_wait_ns(bar, parity, 20000)) {
    if (*c.abort) return false;
    if (clock64() - t0 > kWaitCycles) {
      *c.abort = 1;
      record_fault(c.status, KLC_ERR_DEVICE_TIMEOUT, site, 0);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool wait_bar_short(uint32_t bar, uint32_t parity, const Ctl& c, int site) {
  return mbar_try_wait_ns(bar, parity, 20000) || wait_bar_long(bar, parity, c, site);
}

constexpr int kRows = 128;     // rows of a row tile (TMEM lanes)
constexpr int kKeys = 128;     // keys of a key tile
constexpr int kThreads = 352;  // 8 softmax warps, an MMA warp for each row tile, TMA warp
constexpr int kSoftmaxWarps = 8, kWarpMma0 = 8, kWarpTma = 9, kWarpMma1 = 10;
constexpr uint32_t kTmemCols = 512;
constexpr int kOutPitch = 80, kOutWarp = 32 * kOutPitch;
// A row's reference moves when its maximum has grown by more than 2^kRescale since; it is put 2^kBelow under that maximum,
// so that numerators use f16's range up to 2^15 (bf16: 2^8, no matter).  f16: 2^4 and 2^11; 2^8 would leave 2^7.
template <typename T>
struct Ref {
  static constexpr float kRescale = Elem<T>::kTopLog2 > 0.f ? 4.f : 8.f;
  static constexpr float kBelow = Elem<T>::kTopLog2 > 0.f ? Elem<T>::kTopLog2 - kRescale : 0.f;
};
constexpr int kItems = 2;      // ring of items between the TMA warp and the others

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// waits for the loads into v; the operands keep their uses behind the wait
__device__ __forceinline__ void tmem_wait_ld32(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
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
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float* v) {
  uint32_t r[16];
  tmem_ld16(taddr, r);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, "
      "%44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}

// waits for the loads into v; the operands keep their uses behind the wait
__device__ __forceinline__ void tmem_wait_ld64(float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]), "+r"(r[32]), "+r"(r[33]), "+r"(r[34]), "+r"(r[35]), "+r"(r[36]),
                 "+r"(r[37]), "+r"(r[38]), "+r"(r[39]), "+r"(r[40]), "+r"(r[41]), "+r"(r[42]), "+r"(r[43]),
                 "+r"(r[44]), "+r"(r[45]), "+r"(r[46]), "+r"(r[47]), "+r"(r[48]), "+r"(r[49]), "+r"(r[50]),
                 "+r"(r[51]), "+r"(r[52]), "+r"(r[53]), "+r"(r[54]), "+r"(r[55]), "+r"(r[56]), "+r"(r[57]),
                 "+r"(r[58]), "+r"(r[59]), "+r"(r[60]), "+r"(r[61]), "+r"(r[62]), "+r"(r[63])
               :
               : "memory");
}

// pairs of fp32 in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// 2^x on the FMA pipe, for the share of a tile's exponentials that the special-function unit (16 a clock
// and SM) would be late with.  The range reduction is Cody and Waite's (Software Manual for the Elementary
// Functions, 1980): x = n + f, n the nearest integer (rounded by adding 1.5 * 2^23), n added to the
// exponent.  2^f on [-1/2, 1/2] is the minimax polynomial of the relative error (Chebyshev's alternation;
// a linear programme over 4001 Chebyshev points gives these coefficients to 5e-7): 7.5e-5 with degree 3,
// beside bf16's 2^-8; 2.6e-6 with degree 4, beside f16's 2^-11.  x below -126 counts as -126.
template <typename T>
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  const float2 big = make_float2(12582912.f, 12582912.f);
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 t = add2(x, big);
  const float2 n = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 p;
  if constexpr (Elem<T>::kMmaFormat == 1) {
    p = fma2(f, make_float2(0.05517166802f, 0.05517166802f), make_float2(0.24261112211f, 0.24261112211f));
    p = fma2(f, p, make_float2(0.69326098565f, 0.69326098565f));
    p = fma2(f, p, make_float2(0.99992807355f, 0.99992807355f));
  } else {
    p = fma2(f, make_float2(0.00957010179f, 0.00957010179f), make_float2(0.05591786031f, 0.05591786031f));
    p = fma2(f, p, make_float2(0.24024744831f, 0.24024744831f));
    p = fma2(f, p, make_float2(0.69312181474f, 0.69312181474f));
    p = fma2(f, p, make_float2(0.99999926144f, 0.99999926144f));
  }
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

// D[tmem] (+)= A[tmem or smem] * B[smem].  The whole warp runs these with the same operands and one lane (`lead`)
// issues: operands stay in uniform registers.  Behind a per-lane branch each instruction took
// about 130 cycles to issue, four times what an M = 128, N = 64 product takes to run.
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.u32 e, %6, 0;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 b;\n\t"
      "setp.ne.u32 e, %6, 0;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit_lead(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.u32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(lead)
      : "memory");
}

// fp32 accumulator, both operands of one 16-bit format, A K-major; B K-major or (bit 16) MN-major
template <typename T>
__device__ __forceinline__ constexpr uint32_t f16_idesc(int m, int n, bool b_mn_major) {
  return (1u << 4) | (Elem<T>::kMmaFormat << 7) | (Elem<T>::kMmaFormat << 10) | (b_mn_major ? 1u << 16 : 0u) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

// Shared-memory descriptors with 128-byte swizzle and eight-row groups 1024 bytes apart, as two words; the low word is
// the address and a stride, and only it changes from step to step.  K-major: rows of 64 K elements.  MN-major: rows of
// 64 MN elements, one row per K, the next 64 MN elements `mn_stride` bytes on.
constexpr uint32_t kDescHi = uint32_t(1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t mn_stride) {
  return ((saddr & 0x3FFFFu) >> 4) | ((mn_stride == 0 ? 1u : mn_stride >> 4) << 16);
}

// Whether this lane's share of the rows [from, to) of a value tile holds an element that is not finite; with CLEAR, these
// become 0.
template <typename T, int CHUNKS, bool CLEAR>
__device__ bool odd_rows(unsigned char* v, int from, int to, int lane) {
  constexpr uint32_t kExp = Elem<T>::kMmaFormat == 1 ? 0x7f80u : 0x7c00u;  // all ones: infinite or not a number
  bool some = false;
#pragma unroll 1
  for (int e = from * 8 + lane; e < to * 8; e += 32)
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      uint4* at = reinterpret_cast<uint4*>(v + c * (kKeys * 128) + e * 16);
      uint4 x = *at;
      uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool lo = (w[i] & kExp) == kExp, hi = ((w[i] >> 16) & kExp) == kExp;
        some |= lo | hi;
        if (CLEAR) w[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
      }
      if (CLEAR) *at = x;
    }
  return some;
}

// A value tile whose keys [0, 128) not all rows of the item see, before its product: [first, end) are seen by some row,
// [all_lo, all_end) by all.  A masked weight is 0, and 0 times what is stored must be 0, finite or not:
//   * rows that nobody sees (other sequences', later, windowed out) become zeros;
//   * in rows that some see, elements that are not finite become zeros; `mark` gets `number`, and the rows that see them add them
//     back at the end (add_odd).
// Out of line: it runs on few tiles, and the MMA warp's code is to stay small.  (With two MMA warps both do this, with the same
// result; the mark is there before an element is gone for the other.)
template <typename T, int CHUNKS>
__device__ __noinline__ void settle_values(unsigned char* v, int first, int end, int all_lo, int all_end, volatile uint32_t* mark,
                                           uint32_t number) {
  const int lane = threadIdx.x & 31;
  first = min(max(first, 0), kKeys);
  end = max(min(end, kKeys), first);
  auto zero = [&](int from, int to) {
#pragma unroll 1
    for (int e = from * 8 + lane; e < to * 8; e += 32)
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) *reinterpret_cast<uint4*>(v + c * (kKeys * 128) + e * 16) = make_uint4(0, 0, 0, 0);
  };
  zero(0, first);
  zero(end, kKeys);
  const int a1 = min(all_lo, end), b0 = max(all_end, first);
  const bool some = odd_rows<T, CHUNKS, false>(v, first, a1, lane) | odd_rows<T, CHUNKS, false>(v, b0, end, lane);
  if (__any_sync(0xffffffffu, some)) {
    if (lane == 0) *mark = number;
    __threadfence_block();
    __syncwarp();
    odd_rows<T, CHUNKS, true>(v, first, a1, lane);
    odd_rows<T, CHUNKS, true>(v, b0, end, lane);
  }
  fence_proxy_async();
  __syncwarp();
}

struct Item {
  int q0, qn;  // the sequence's first query row and its number of query rows (tokens)
  int k0, kn;  // first key row and number of keys
  int tok0;    // first token of the item's row tiles; -1: no more items
  int tiles;   // row tiles with rows: 1 or 2
  int lo, n;   // first key of the item's tiles, and their number
  int kvh, z;  // key head; prefix: share of the keys
  int first, last;  // lowest and highest key that some row of the item sees
  int all_lo, all_hi;  // every row sees the keys from all_lo to all_hi
};

template <int D>
struct Cfg {
  static constexpr int kChunks = D / 64;                    // 128-byte columns of a head's row
  static constexpr int kTile = kKeys * D * 2;               // bytes of a query, key or value tile
  static constexpr int kStages = D == 64 ? 5 : 2;           // ring of key and value tiles: 160 / 128 KB
  // of 8 pairs of exponentials, on the FMA pipe: 6016 tokens ran at 643 / 654 / 706 / 690 TFLOP/s with 0 / 1 / 2 / 3
  // (D = 64), 958 / 970 / 986 / 976 (D = 128)
  static constexpr int kFmaPairs = 2;
  // TMEM columns: S 0-255, O behind it.  D = 64 leaves room for P, so the next S can be made while this one's
  // exponentials are; with D = 128 P lies over the upper half of S, which is in registers by then.
  static constexpr bool kOwnP = D == 64;
  static constexpr int kMmaWarps = kOwnP ? 2 : 1;
  static constexpr int kColO = 2 * kKeys;
  static constexpr int kColP = kOwnP ? kColO + 2 * D : kKeys / 2, kStepP = kOwnP ? kKeys / 2 : kKeys;
  static constexpr int OFF_Q = 0;                           // two row tiles
  static constexpr int OFF_KV = 2 * kTile;
  static constexpr int OFF_BAR = OFF_KV + kStages * 2 * kTile;
  static constexpr int kBars = 2 * kStages + 2 + 10 + 2 * kItems + 1;
  static constexpr int OFF_MISC = OFF_BAR + kBars * 8;
  static constexpr int OFF_ITEM = OFF_MISC + 32;
  static constexpr int OFF_RECENT = OFF_ITEM + kItems * int(sizeof(Item));  // the last four items
  static constexpr int OFF_OUT = (OFF_RECENT + 4 * int(sizeof(Item)) + 15) / 16 * 16;  // per softmax warp: 32 rows of 64 + 16 bytes
  static constexpr int kSmem = OFF_OUT + (D == 128 ? kSoftmaxWarps * kOutWarp : 0) + 1024;  // + alignment of the swizzled tiles
};

// Adds to a row's output in TMEM what odd_rows took out of the values: the elements that are not finite of those keys of the
// item's tiles that the row, but not every row of the item, sees (a positive weight times an infinity or a NaN is that).
template <typename T, int D, bool PREFIX>
__device__ __noinline__ void add_odd(uint32_t o_col, const Item& it, const TcParams& p, int jlo, int jhi) {
  for (int c = 0; c < D / 32; ++c) {
    float o[32];
    tmem_ld32(o_col + uint32_t(32 * c), o);
    tmem_wait_ld32(o);
    for (int j = max(max(it.first, it.lo), jlo); j <= min(min(it.last, it.lo + it.n * kKeys - 1), jhi); ++j) {
      if (j >= it.all_lo && j <= it.all_hi) {
        j = it.all_hi;
        continue;
      }
      const T* v = reinterpret_cast<const T*>(p.v) + 32 * c;
      if (PREFIX) {
        const int page = p.block_table[int64_t(it.q0) * p.table_stride + j / p.page_size];
        if (page < 0 || page >= p.pages) continue;
        v += page * p.v_ts + (int64_t(it.kvh) * p.page_size + j % p.page_size) * D;
      } else {
        v += (int64_t(it.k0) + j) * p.v_ts + int64_t(it.kvh) * p.v_hs;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 x = Elem<T>::unpack(*reinterpret_cast<const uint32_t*>(v + e));
        if (!isfinite(x.x)) o[e] += x.x;
        if (!isfinite(x.y)) o[e + 1] += x.y;
      }
    }
    __syncwarp();
    tmem_st32(o_col + uint32_t(32 * c), reinterpret_cast<const uint32_t*>(o));
  }
  tmem_wait_st();
}

// Records the table entries of the prefix's keys [from, to) that are no page of the pool, where one of `rows` rows sees a key of
// the page: windows of rows of very different lengths leave pages between them that no row sees, whose entries may be gone.
// (Behind the loads of an item that met such an entry; 64 rows behind 16384 keys: 54.2 us, 56.7 with a call in their loop.)
__device__ __noinline__ void report_pages(const TcParams& p, const int32_t* table, const int32_t* lens, int rows, int keys, int from, int to) {
  for (int key = from / p.page_size * p.page_size; key < to; key += p.page_size) {
    const int page = table[key / p.page_size];
    if (page >= 0 && page < p.pages) continue;
    for (int i = 0; i < rows; ++i)
      if (min(lens[i], keys) > key && (p.window > 0 ? max(0, lens[i] - p.window) : 0) < key + p.page_size) {
        record_fault(p.status, KLC_ERR_DEVICE_FAULT, 521, page);
        return;
      }
  }
}

// ---------------------------------------------------------------------------
// PREFIX = false: packed prompts.  PREFIX = true: single-token rows over the pages of their group's prefix, keys
// split `splits` ways; shares (m, l, o) go to the workspace and are joined by the decode join.
//
// Persistent: CTA c takes the items c, 2N - 1 - c, 2N + c, ... (back and forth, so that with items in
// descending size no CTA gets the large end of every wave).  The TMA warp finds the items and hands them
// to the others through a small ring, so the next item's loads and first S run under this one's tail.
// ---------------------------------------------------------------------------
template <typename T, int D, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcParams p) {
  using C = Cfg<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int G = p.group, tpt = p.tpt;

  const uint32_t bar0 = smem_u32(smem + C::OFF_BAR);
  auto kv_full = [&](int s) { return bar0 + 8u * s; };
  auto kv_empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };
  constexpr int kB = 2 * C::kStages;
  const uint32_t q_full = bar0 + 8u * kB, q_empty = bar0 + 8u * (kB + 1);
  auto s_full = [&](int t) { return bar0 + 8u * (kB + 2 + t); };
  auto p_full = [&](int t) { return bar0 + 8u * (kB + 4 + t); };
  auto o_full = [&](int t) { return bar0 + 8u * (kB + 6 + t); };
  auto s_free = [&](int t) { return bar0 + 8u * (kB + 8 + t); };
  auto p_half = [&](int t) { return bar0 + 8u * (kB + 10 + t); };
  auto item_full = [&](int i) { return bar0 + 8u * (kB + 12 + i); };
  auto item_empty = [&](int i) { return bar0 + 8u * (kB + 12 + kItems + i); };
  const uint32_t mma_done = bar0 + 8u * (kB + 12 + 2 * kItems);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::OFF_MISC + 4);
  // [4]: number of the last item (+ 1, by item number mod 4) in which a value that only some rows see was not finite
  volatile uint32_t* odd = reinterpret_cast<volatile uint32_t*>(smem + C::OFF_MISC + 8);
  Item* recent = reinterpret_cast<Item*>(smem + C::OFF_RECENT);
  Item* items = reinterpret_cast<Item*>(smem + C::OFF_ITEM);
  const Ctl ctl{abort_flag, p.status};

  if (tid == 32 * kWarpTma) {
    prefetch_map(&map_q);
    prefetch_map(&map_k);
    prefetch_map(&map_v);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), C::kMmaWarps);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, C::kMmaWarps);
    for (int t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t), kRows);
      mbar_init(p_half(t), kRows);
      mbar_init(s_free(t), kRows);
      mbar_init(o_full(t), 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(item_full(i), 1);
      mbar_init(item_empty(i), kSoftmaxWarps + C::kMmaWarps);
    }
    mbar_init(mma_done, C::kMmaWarps);
    *abort_flag = 0;
    for (int i = 0; i < 4; ++i) odd[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kWarpMma0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);
  pdl_wait();     // set up under the previous kernel's tail; from here on its results are read
  pdl_trigger();  // the next kernel may set up meanwhile (prefix: the decode kernel may run beside this one)

  // the next item of the ring for a consumer warp; false after the last one or on an abort
  uint32_t item_no = 0;
  auto next_item = [&](Item* it, int site) {
    const int s = item_no % kItems;
    bool ok = wait_bar_short(item_full(s), (item_no / kItems) & 1, ctl, site);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) *it = items[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(item_empty(s));
    ++item_no;
    return ok && it->tok0 >= 0;
  };

  if (warp == kWarpTma) {
    // ---------------------------------------------------------------- items and loads
    int seq0 = 0;        // sequences before this one are done with
    int64_t base = 0;    // row-tile pairs before sequence seq0
    const int unit = p.kv_heads * (PREFIX ? p.splits : 1);  // items of a pair
    uint32_t issued = 0, queries = 0;
    bool ok = true;
    for (uint32_t wave = 0; ok; ++wave) {
      const int64_t idx = int64_t(wave) * gridDim.x + ((wave & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
      const int64_t pair = idx / unit;
      const int sub = int(idx - pair * unit);
      Item it{0, 0, 0, 0, -1, 0, 0, 0, 0, 0, 0, 0, 0, 0};
      for (; seq0 < p.batch; seq0 += 32) {
        const int s = seq0 + lane;
        int qb = 0, qn = 0, kb = 0, kn = 0;
        if (s < p.batch) {
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
        const int pairs = int((int64_t(qn) + 2 * tpt - 1) / (2 * tpt));
        int incl = pairs;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += v;
        }
        const int64_t excl = base + incl - pairs;
        const bool mine = pair >= excl && pair < excl + pairs;
        const unsigned hit = __ballot_sync(0xffffffffu, mine);
        if (hit != 0) {
          const int src = __ffs(hit) - 1;
          it.q0 = __shfl_sync(0xffffffffu, qb, src);
          it.qn = __shfl_sync(0xffffffffu, qn, src);
          it.k0 = __shfl_sync(0xffffffffu, kb, src);
          it.kn = __shfl_sync(0xffffffffu, kn, src);
          // a sequence's last rows see the most keys: its tiles run in descending order
          it.tok0 = __shfl_sync(0xffffffffu, (pairs - 1 - int(pair - excl)) * 2 * tpt, src);
          break;
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (it.tok0 >= 0) {
        it.kvh = PREFIX ? sub / p.splits : sub;
        it.z = PREFIX ? sub - it.kvh * p.splits : 0;
        it.tiles = it.tok0 + tpt < it.qn ? 2 : 1;
        int first, last;  // keys some row of the item sees
        if (PREFIX) {
          // over the rows that see keys of the prefix at all: an idle row would make every tile a boundary one
          int lo_min = 0x7fffffff, lo_max = 0, hi_min = 0x7fffffff, hi_max = -1;
          for (int i = it.tok0 + lane; i < min(it.tok0 + 2 * tpt, it.qn); i += 32) {
            const int len = p.lens[it.q0 + i], lo = p.window > 0 ? max(0, len - p.window) : 0, hi = min(len, it.kn) - 1;
            if (lo > hi) continue;
            lo_min = min(lo_min, lo);
            lo_max = max(lo_max, lo);
            hi_min = min(hi_min, hi);
            hi_max = max(hi_max, hi);
          }
          first = __reduce_min_sync(0xffffffffu, lo_min);
          last = __reduce_max_sync(0xffffffffu, hi_max);
          it.all_lo = __reduce_max_sync(0xffffffffu, lo_max);
          it.all_hi = __reduce_min_sync(0xffffffffu, hi_min);
        } else {
          const int pos = it.kn - it.qn + it.tok0;
          first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
          last = it.kn - it.qn + min(it.tok0 + 2 * tpt, it.qn) - 1;
          it.all_lo = p.window > 0 ? max(0, last - p.window + 1) : 0;
          it.all_hi = pos;
        }
        if (PREFIX) {  // this item's share of the tiles, which start where pages do
          int lo = 0, n = 0;
          if (last >= first) lo = first / kKeys, n = last / kKeys + 1 - lo;
          const int a = int(int64_t(n) * it.z / p.splits);
          it.lo = (lo + a) * kKeys;
          it.n = int(int64_t(n) * (it.z + 1) / p.splits) - a;
        } else if (last >= first) {
          it.lo = first;
          it.n = (last - first) / kKeys + 1;
        }
        it.first = first;
        it.last = last;
      }
      const int slot = wave % kItems;
      ok = wait_bar_short(item_empty(slot), ((wave / kItems) & 1) ^ 1, ctl, 510);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      if (lane == 0) {
        items[slot] = it;
        recent[wave & 3] = it;
        mbar_arrive(item_full(slot));
      }
      if (it.tok0 < 0) break;
      if (lane == 0) {
        bool no_page = false;  // prefix: an entry that is no page of the pool
        for (int i = 0; i < it.n; ++i, ++issued) {
          const int key = it.lo + i * kKeys, s = issued % C::kStages;
          if (!(ok = wait_bar_short(kv_empty(s), ((issued / C::kStages) & 1) ^ 1, ctl, 501))) break;
          mbar_arrive_expect_tx(kv_full(s), 2u * uint32_t(C::kTile));
          for (int kv = 0; kv < 2; ++kv) {
            const uint32_t dst = smem_u32(smem + C::OFF_KV + (2 * s + kv) * C::kTile);
            const CUtensorMap* map = kv ? &map_v : &map_k;
            if (!PREFIX) {
              for (int c = 0; c < C::kChunks; ++c)
                tma_load_3d(dst + c * (kKeys * 128), map, c * 64, it.kvh, it.k0 + key, kv_full(s));
            } else {
              // pages without a key that some row sees (their entries may be gone), and ids that are no page of the pool, read
              // as zeros (coordinate past the end)
              for (int j = 0; j < kKeys; j += p.page_size) {
                int page = int(p.pages);
                if (key + j <= it.last && key + j + p.page_size > it.first) {
                  page = p.block_table[int64_t(it.q0) * p.table_stride + (key + j) / p.page_size];
                  if (page < 0 || page >= p.pages) {
                    no_page = true;
                    page = int(p.pages);
                  }
                }
                for (int c = 0; c < C::kChunks; ++c)
                  tma_load_4d(dst + c * (kKeys * 128) + j * 128, map, c * 64, 0, it.kvh, page, kv_full(s));
              }
            }
          }
          if (i == 0) {  // the item's queries, behind its first keys: they wait for the previous item's last S
            if (!(ok = wait_bar_short(q_empty, (queries & 1) ^ 1, ctl, 511))) {
              ++issued;
              break;
            }
            mbar_arrive_expect_tx(q_full, uint32_t(it.tiles * C::kChunks * tpt * G) * 128u);
            for (int tt = 0; tt < it.tiles; ++tt)
              for (int c = 0; c < C::kChunks; ++c)
                tma_load_3d(smem_u32(smem + C::OFF_Q + tt * C::kTile + c * (kRows * 128)), &map_q, c * 64, it.kvh * G,
                            it.q0 + it.tok0 + tt * tpt, q_full);
            ++queries;
          }
        }
        if (PREFIX && no_page)
          report_pages(p, p.block_table + int64_t(it.q0) * p.table_stride, p.lens + it.q0 + it.tok0, min(2 * tpt, it.qn - it.tok0), it.kn,
                       max(it.first, it.lo), min(it.last + 1, it.lo + it.n * kKeys));
      }
      ok = __shfl_sync(0xffffffffu, int(ok), 0) != 0;
    }
    if (!ok && lane == 0) {
      if (queries > 0) drain_wait(q_full, (queries - 1) & 1);
      drain_ring(kv_full(0), C::kStages, issued);
    }
    __syncwarp();
  } else if (warp == kWarpMma0 || (warp == kWarpMma1 && C::kMmaWarps == 2)) {
    // ---------------------------------------------------------------- MMA
    // D = 64: one warp per row tile, so that neither tile's chain waits behind the other's in program order.  D = 128: one
    // warp for both, in turns: a tile's P V and next S run as one block of the tensor pipe while the other tile is in its
    // softmax (issued side by side, the two tiles fell into step and tensor pipe and softmax idled in turns: 812 against 1025
    // TFLOP/s).  Little code: this warp's instructions are evicted from the cache by the softmax warps' between its turns.
    constexpr uint32_t idesc_qk = f16_idesc<T>(kRows, kKeys, false);
    constexpr uint32_t idesc_pv = f16_idesc<T>(kRows, D, true);
    constexpr uint32_t kTileLo = C::kTile >> 4;  // a tile in descriptor units
    constexpr int kMine = 3 - C::kMmaWarps;      // row tiles of this warp
    const int t0 = warp == kWarpMma0 ? 0 : 1;
    bool ok = true;
    uint32_t lead;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(lead));
    auto wait_all = [&](uint32_t bar, uint32_t parity, int site) {
      const bool w = wait_bar_short(bar, parity, ctl, site);
      return __all_sync(0xffffffffu, w) != 0;
    };
    const uint32_t q_lo = desc_lo(smem_u32(smem + C::OFF_Q), 0), k_lo = desc_lo(smem_u32(smem + C::OFF_KV), 0);
    const uint32_t v_lo = desc_lo(smem_u32(smem + C::OFF_KV), kKeys * 128) + kTileLo;
    // ring cursors of the next S and of the next product (one stage behind), with phase parities
    uint32_t ck = 0, ck_ph = 0, cv = 0;
    auto advance = [](uint32_t c) { return c + 1 == uint32_t(C::kStages) ? 0u : c + 1; };
    uint32_t queries = 0, step[2] = {0, 0};
    Item it;
    while (ok && next_item(&it, 512)) {
      const int n = it.n, mine = min(kMine, it.tiles - t0);
      if (n == 0) continue;
      if (mine <= 0) {  // no row in this warp's tile: pass the stages and the queries on
        for (int i = 0; i < n && ok; ++i) {
          if (!(ok = wait_all(kv_full(ck), ck_ph, 503))) break;
          if (lane == 0) mbar_arrive(kv_empty(ck));
          ck = advance(ck);
          ck_ph ^= ck == 0;
        }
        cv = ck;
        if (ok && (ok = wait_all(q_full, queries & 1, 502)) && lane == 0) mbar_arrive(q_empty);
        __syncwarp();
        ++queries;
        continue;
      }
      // S = Q K^T for step i + 1 of this warp's j-th row tile, once S is free: read by its softmax (D = 64), or behind the
      // P V that read P from it (issue order, D = 128)
      auto next_s = [&](int i, int j) {
        if (i + 1 >= n) return true;
        const int tt = t0 + j;
        if (j == 0 && !wait_all(kv_full(ck), ck_ph, 503)) return false;
        if (j == 0 && i < 0 && !wait_all(q_full, queries & 1, 502)) return false;
        if (C::kOwnP && step[j] + (i >= 0) > 0 && !wait_all(s_free(tt), (step[j] + (i >= 0) + 1) & 1, 514)) return false;
        tc_fence_after();
        const uint32_t a = q_lo + uint32_t(tt) * kTileLo, b = k_lo + ck * (2 * kTileLo);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = uint32_t((kk >> 2) * (kRows * 128) + (kk & 3) * 32) >> 4;
          mma_ss(lead, tmem + uint32_t(tt * kKeys), a + off, b + off, kDescHi, idesc_qk, kk > 0);
        }
        commit_lead(lead, s_full(tt));
        if (j + 1 == mine) {
          if (i + 2 == n) commit_lead(lead, q_empty);
          ck = advance(ck);
          ck_ph ^= ck == 0;
        }
        return true;
      };
      auto product = [&](int i, int j) {  // O += P V of step i
        if (i < 0) return true;
        const int tt = t0 + j;
        const int key = it.lo + i * kKeys;
        if (j == 0 && (key < it.all_lo || key + kKeys - 1 > it.all_hi)) {
          settle_values<T, C::kChunks>(smem + C::OFF_KV + (2 * cv + 1) * C::kTile, it.first - key, it.last + 1 - key, it.all_lo - key,
                                       it.all_hi + 1 - key, &odd[(item_no - 1) & 3], item_no);
        }
        const uint32_t b = v_lo + cv * (2 * kTileLo);
        auto keys64 = [&](int k0, bool first) {
#pragma unroll
          for (int kk = k0; kk < k0 + kKeys / 32; ++kk)
            mma_ts(lead, tmem + uint32_t(C::kColO + tt * D), tmem + uint32_t(C::kColP + tt * C::kStepP + kk * 8),
                   b + uint32_t(kk * 16 * 128 >> 4), kDescHi, idesc_pv, kk > k0 || !first);
        };
        if (!C::kOwnP) {  // P comes in two halves, keys 64-127 first
          if (!wait_all(p_half(tt), step[j] & 1, 515)) return false;
          tc_fence_after();
          keys64(4, i == 0);
        }
        if (!wait_all(p_full(tt), step[j] & 1, 505)) return false;
        tc_fence_after();
        if (C::kOwnP) keys64(4, i == 0);
        keys64(0, false);
        commit_lead(lead, o_full(tt));
        if (j + 1 == mine) {
          commit_lead(lead, kv_empty(cv));
          cv = advance(cv);
        }
        ++step[j];
        return true;
      };
      // step -1 makes the first S, step i the next one and this step's product
#pragma unroll 1
      for (int i = -1; i < n && ok; ++i) {
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          if (!ok || j >= mine) break;
          if constexpr (C::kOwnP) ok = next_s(i, j) && product(i, j);
          else ok = product(i, j) && next_s(i, j);
        }
      }
      ++queries;
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {  // no MMA may still be in flight when TMEM is freed
      commit_lead(lead, mma_done);
      if (lane == 0) drain_wait(mma_done, 0);
      __syncwarp();
    }
  } else if (warp < kSoftmaxWarps) {
    // ---------------------------------------------------------------- softmax
    const int t = warp >> 2;  // row tile
    const int r = tid & (kRows - 1);
    const int tok_in = r / G, g = r - tok_in * G;
    const uint32_t lane_base = uint32_t((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lane_base + uint32_t(t * kKeys);
    const uint32_t o_col = tmem + lane_base + uint32_t(C::kColO + t * D);
    const uint32_t p_col = tmem + lane_base + uint32_t(C::kColP + t * C::kStepP);
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    uint32_t steps = 0;
    Item it;
    while (next_item(&it, 513)) {
      if (t >= it.tiles) continue;  // no row in this tile
      // the row and the keys [jlo, jhi] it sees
      const int tok = it.tok0 + t * tpt + tok_in;
      const bool row_ok = r < tpt * G && tok < it.qn;
      int jlo = 0x7fffffff, jhi = -1;
      if (row_ok) {
        const int pos = PREFIX ? p.lens[it.q0 + tok] - 1 : it.kn - it.qn + tok;
        jhi = PREFIX ? min(pos, it.kn - 1) : pos;
        jlo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        if (jlo > jhi) jlo = 0x7fffffff, jhi = -1;
      }
      // the row reaches these tiles whole: rows that are not there do not make a tile a boundary one (nor do, in a prefix, rows
      // that see none of it: they keep m = -inf, a share that the join leaves out whatever its O holds)
      const bool live = PREFIX ? row_ok && jhi >= 0 : row_ok;
      const int wlo = __reduce_max_sync(0xffffffffu, live ? jlo : 0), whi = __reduce_min_sync(0xffffffffu, live ? jhi : 0x7fffffff);
      const int head = it.kvh * G + g;
      const float sink = !PREFIX && row_ok && p.sinks != nullptr ? p.sinks[head] * kLog2e : 0.f;  // used at the end
      float m = -INFINITY, l = 0.f;  // m: reference (log2 units) of the stored P and O
      bool ok = true;
      for (int i = 0; i < it.n; ++i, ++steps) {
        ok = wait_bar_short(s_full(t), steps & 1, ctl, 508);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
        const int kb = it.lo + i * kKeys;
        const bool masked = kb < wlo || kb + kKeys - 1 > whi;
        const int ja = jlo - kb, jb = jhi - kb;
        // Columns 0-63 are read twice and 64-127 kept (all 128 would not fit the registers).
        float sa[64], sb[64];
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        tmem_ld64(s_col, sa);
        tmem_wait_ld64(sa);
        tmem_ld64(s_col + 64, sb);
        // boundary tiles, 32 columns at a time: bit c, no row of the warp sees any / some row does not see all of columns 32 c ..
        // (D = 64: 2 to 6 % faster on ragged and windowed prompts; with D = 128 2 % slower, by registers)
        uint32_t none = 0, part = masked ? 15u : 0u;
        if (C::kOwnP && masked) {
          part = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (!__any_sync(0xffffffffu, ja <= 32 * c + 31 && jb >= 32 * c)) none |= 1u << c;
            if (__any_sync(0xffffffffu, live && (ja > 32 * c || jb < 32 * c + 31))) part |= 1u << c;
          }
          part &= ~none;
        }
        auto hide = [&](float* s, int c) {
          if (part >> c & 1) {
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = (32 * c + j >= ja && 32 * c + j <= jb) ? s[j] : -INFINITY;
          } else if (none >> c & 1) {
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = -INFINITY;
          }
        };
        auto peak = [&](const float* s) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) mx[(j >> 1) & 3] = max3_nan(mx[(j >> 1) & 3], s[j], s[j + 1]);
        };
        if (masked) {
          hide(sa, 0);
          hide(sa + 32, 1);
        }
        peak(sa);
        peak(sa + 32);
        tmem_wait_ld64(sb);
        if (masked) {
          hide(sb, 2);
          hide(sb + 32, 3);
        }
        peak(sb);
        peak(sb + 32);
        const float top = max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2 - Ref<T>::kBelow;
        // the reference moves when the maximum has grown by more than 2^kRescale, or to a NaN, and stays there: a tile without
        // keys must not take its place
        const bool grow = live && (m == -INFINITY ? top != -INFINITY : top > m + Ref<T>::kRescale || top != top);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? (m == -INFINITY ? 0.f : exp2_approx(m - top)) : 1.f;
          if (grow) {
            m = top == INFINITY ? __int_as_float(0x7fffffff) : top;  // inf - inf is not a number; the FMA pipe's share would hide it
            l *= f;
          }
          // O is complete behind the previous P V (D = 128: S of this tile was issued behind it)
          if (C::kOwnP && i > 0) {
            ok = wait_bar_short(o_full(t), (steps - 1) & 1, ctl, 516);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
          }
          if (i > 0) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              float o[16];
              tmem_ld16f(o_col + uint32_t(16 * c), o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] *= f;
              tmem_st16(o_col + uint32_t(16 * c), reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
        float s0[32];
        tmem_ld32(s_col, s0);
        const float mref = m == -INFINITY ? 0.f : m;
        const float2 off2 = make_float2(-mref, -mref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        // numerators of 32 scores, packed; boundary tiles use the special-function unit alone (it gives an exact 0)
        auto numerators = [&](const float* s, uint32_t* pk, auto whole) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 x = fma2(make_float2(s[j], s[j + 1]), scale2, off2);
            float2 e;
            if (decltype(whole)::value && (j >> 1) % 8 < C::kFmaPairs) e = exp2_fma<T>(x);
            else e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
            sum[(j >> 1) & 1] = add2(sum[(j >> 1) & 1], e);
            pk[j >> 1] = Elem<T>::pack(e.x, e.y);
          }
        };
        auto write_p = [&](auto whole) {
          auto hide_again = [&](float* s, int c) {
            if (!decltype(whole)::value) hide(s, c);
          };
          if constexpr (C::kOwnP) {
            uint32_t pk[32];
            numerators(sb, pk, whole);
            numerators(sb + 32, pk + 16, whole);
            tmem_wait_ld32(s0);
            float s1[32];
            tmem_ld32(s_col + 32, s1);
            if (i > 0) {  // the previous P V still reads P till then
              ok = wait_bar_short(o_full(t), (steps - 1) & 1, ctl, 517);
              ok = __all_sync(0xffffffffu, ok);
              tc_fence_after();
            }
            tmem_st32(p_col + 32, pk);
            hide_again(s0, 0);
            numerators(s0, pk, whole);
            tmem_wait_ld32(s1);
            tc_fence_before();
            mbar_arrive(s_free(t));
            hide_again(s1, 1);
            numerators(s1, pk + 16, whole);
            tmem_st32(p_col, pk);
          } else {
            uint32_t pk[16];
            numerators(sb, pk, whole);
            tmem_st16(p_col + 32, pk);
            tmem_wait_ld32(s0);
            numerators(sb + 32, pk, whole);
            tmem_st16(p_col + 48, pk);
            float s1[32];
            tmem_ld32(s_col + 32, s1);
            tmem_wait_st();  // keys 64-127: their half of the product starts here
            tc_fence_before();
            mbar_arrive(p_half(t));
            hide_again(s0, 0);
            numerators(s0, pk, whole);
            tmem_st16(p_col, pk);
            tmem_wait_ld32(s1);
            hide_again(s1, 1);
            numerators(s1, pk, whole);
            tmem_st16(p_col + 16, pk);
          }
        };
        if (masked) write_p(std::false_type{});
        else write_p(std::true_type{});
        const float2 both = add2(sum[0], sum[1]);
        l += both.x + both.y;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_full(t));
        if (!ok) break;
      }
      // ---- epilogue: the row's output
      if (ok && it.n > 0) {
        ok = wait_bar_short(o_full(t), (steps - 1) & 1, ctl, 509);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (!ok) break;
      if (m == -INFINITY) l = 0.f;  // no key, or scores of -inf alone (the FMA pipe's share of a whole tile is not an exact 0)
      const int64_t row = int64_t(it.q0) + tok;
      if (odd[(item_no - 1) & 3] == item_no) add_odd<T, D, PREFIX>(o_col, recent[(item_no - 1) & 3], p, jlo, jhi);
      if (PREFIX) {
        const int64_t slot = (int64_t(it.z) * p.total_q + row) * p.heads + head;
        if (row_ok) p.part_ml[slot] = make_float2(m, l);
        if (it.n > 0) {
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
        float inv = 0.f, lse = 0.f;
        if (row_ok) {
          finish_row(m, l, p.sinks != nullptr, sink, &inv, &lse);
          if (p.lse != nullptr) p.lse[row * p.heads + head] = lse;
        }
        // D = 128: through shared memory, 32 columns at a time, so that four lanes store 64 bytes of a row (1106 against 1067
        // TFLOP/s at 6016 tokens); D = 64: straight from the rows' threads (718 against 678).
        if constexpr (D == 128) {
          const int64_t mine = row_ok ? row * p.out_ts + int64_t(head) * p.out_hs : -1;
          int64_t off[4];  // of the rows this lane stores: 8 k + lane / 4 of the warp's
#pragma unroll
          for (int k = 0; k < 4; ++k) off[k] = __shfl_sync(0xffffffffu, mine, 8 * k + (lane >> 2));
          unsigned char* stage = smem + C::OFF_OUT + warp * kOutWarp;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            if (it.n > 0) {
              tmem_ld32(o_col + uint32_t(32 * c), o);
              tmem_wait_ld32(o);
              } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint4 w;
              w.x = Elem<T>::pack(o[8 * j] * inv, o[8 * j + 1] * inv);
              w.y = Elem<T>::pack(o[8 * j + 2] * inv, o[8 * j + 3] * inv);
              w.z = Elem<T>::pack(o[8 * j + 4] * inv, o[8 * j + 5] * inv);
              w.w = Elem<T>::pack(o[8 * j + 6] * inv, o[8 * j + 7] * inv);
              *reinterpret_cast<uint4*>(stage + lane * kOutPitch + 16 * j) = w;
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint4 w = *reinterpret_cast<const uint4*>(stage + (8 * k + (lane >> 2)) * kOutPitch + (lane & 3) * 16);
              if (off[k] >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + off[k] + 32 * c + (lane & 3) * 8) = w;
            }
            __syncwarp();
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row * p.out_ts + int64_t(head) * p.out_hs);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            if (it.n > 0) {
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
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
}

template <typename T, int D, bool PREFIX>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TcParams& p, int64_t items, cudaStream_t s) {
  auto kernel = attn_tc_kernel<T, D, PREFIX>;
  static SmemLimit limit;
  int st = limit.raise(reinterpret_cast<const void*>(kernel), Cfg<D>::kSmem);
  if (st != KLC_OK) return st;
  KLC_CUDA(launch_chain(kernel, dim3(unsigned(std::min<int64_t>(items, sm_count()))), dim3(kThreads), Cfg<D>::kSmem, s, 0, mq, mk, mv, p));
  KLC_LAUNCH_CHECK(PREFIX ? "attn_prefix" : "attn_prompt");
  return KLC_OK;
}

template <bool PREFIX>
int launch_typed(int dtype, int head_dim, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
                 const TcParams& p, int64_t items, cudaStream_t s) {
  if (dtype == KLC_BF16)
    return head_dim == 64 ? launch<__nv_bfloat16, 64, PREFIX>(mq, mk, mv, p, items, s)
                          : launch<__nv_bfloat16, 128, PREFIX>(mq, mk, mv, p, items, s);
  return head_dim == 64 ? launch<__half, 64, PREFIX>(mq, mk, mv, p, items, s) : launch<__half, 128, PREFIX>(mq, mk, mv, p, items, s);
}

CUtensorMapDataType map_type(int dtype) {
  return dtype == KLC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// rows [tokens][heads][D] with token / head strides in elements; box of `box_heads` x `box_tokens`
int rows_map(CUtensorMap* m, int dtype, int head_dim, const void* base, int64_t tokens, int heads, int64_t ts, int64_t hs,
             int box_heads, int box_tokens) {
  // the stride of a dimension of one means nothing, but the map wants one
  if (heads == 1) hs = head_dim;
  if (tokens <= 1) ts = hs * heads;
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
  p.kv_heads = d.kv_heads;
  p.splits = d.splits;
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
  p.v = v_pages;
  p.v_ts = page_stride;
  p.part_o = d.prefix_o;
  p.part_ml = d.prefix_ml;
  CUtensorMap mq, mk, mv;
  int st = rows_map(&mq, dims.dtype, dims.head_dim, q, d.batch, d.heads, d.q_ts, d.q_hs, d.group, p.tpt);
  if (st == KLC_OK) st = pool_map(&mk, dims.dtype, dims.head_dim, k_pages, d.pages, d.kv_heads, d.page_size, page_stride, d.page_size);
  if (st == KLC_OK) st = pool_map(&mv, dims.dtype, dims.head_dim, v_pages, d.pages, d.kv_heads, d.page_size, page_stride, d.page_size);
  if (st != KLC_OK) return st;
  const int tok = 2 * p.tpt;
  const int pairs = d.groups == 1 ? (d.batch + tok - 1) / tok : std::min(d.batch, d.batch / tok + d.groups);
  return launch_typed<true>(dims.dtype, dims.head_dim, mq, mk, mv, p, int64_t(pairs) * d.kv_heads * d.splits, stream);
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
  p.kv_heads = dims->kv_heads;
  p.group = G;
  p.tpt = kRows / G;
  p.scale_log2 = dims->scale * kLog2e;
  p.v = v;
  p.v_ts = v_token_stride;
  p.v_hs = v_head_stride;
  p.window = std::min(dims->window, 1 << 30);  // no position is larger, and position - window stays in 32 bits
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
  return launch_typed<false>(dims->dtype, d, mq, mk, mv, p, gx * dims->kv_heads, as_stream(stream));
}
