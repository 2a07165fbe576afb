// What the tensor-core kernels of attention inside packed structures share: operand tiles, descriptors, barriers, tensor memory.
//
// An operand tile is 128 rows of up to 64 values (64 or 128 bytes a row, swizzled), several of them side by side (Geometry), brought in by TMA
// from the strided operand: a map has the dimensions (values, rows, heads), values behind the last one come as zeros.  The same image serves the tensor cores with d contracted (K-major) and with the rows contracted (MN-major), so a tile of keys
// serves q k^T and dS k, a tile of queries k q^T and dS^T q.  A tile may reach over the end of its structure into the next one's rows: where
// they would be contracted, the loading warp clears them before it hands the tile over (a zero probability times a neighbour's NaN is NaN).
#pragma once
#include <cuda.h>

#include "packed_mma.cuh"

namespace so3lr {
namespace tc {

using packed::smem_addr;

constexpr int kTile = 128;
constexpr int kMmaWarp = 8, kLoadWarp = 9;      // 0 .. 7 compute, 10 and 11 fetch statistics in the kernel of dk and dv
constexpr int kThreads = 384;
// registers a thread of the compute and of the other warps after the split: 256 x 208 + 128 x 88 = 384 x 168, the launch's total
constexpr int kComputeRegs = 208, kOtherRegs = 88;
constexpr int kEndTries = 2000000;      // 8 s

// holds the thread for up to some 4 us
__device__ __forceinline__ bool test_bar(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Every wait ends: after `tries` tries, or when another one of this CTA has run out.  From then on no copy is issued, jobs are passed on without
// tiles and their rows written as NaN, and the CTA ends behind what is under way (end), where it tells the host (report).  What stands in a wait
// shows: with the first try as one of the loop's dk and dv of 8,192 rows, 9 x 64, take 364 us instead of 351, with a clock in the loop the forward
// kernel of 24 structures of 150 to 900 rows 99 instead of 92.
struct Wait {
  uint32_t failed_at;        // the word of shared memory that says so
  int tries;
  __device__ __forceinline__ bool failed() const {
    uint32_t x;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(x) : "r"(failed_at) : "memory");
    return x != 0;
  }
  __device__ __forceinline__ void fail() const { asm volatile("st.volatile.shared.u32 [%0], 1;" ::"r"(failed_at) : "memory"); }
  __device__ __forceinline__ bool operator()(uint32_t bar, uint32_t parity) const {
    if (test_bar(bar, parity)) return true;
    for (int left = tries; --left >= 0 && !failed();)
      if (test_bar(bar, parity)) return true;
    fail();
    return false;
  }
  // The loading warp's.  With negative tries, for tests, what is not over at once has run out.
  __device__ __forceinline__ bool of_loader(uint32_t bar, uint32_t parity) const {
    if (tries >= 0) return (*this)(bar, parity);
    uint32_t now;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(now) : "r"(bar), "r"(parity) : "memory");
    if (!now) fail();
    return now != 0;
  }
  // The waits that hold after a failure too: for what is under way, and for the next job.  What they wait for comes once the waits above have
  // ended; kEndTries is the bound for what should not be.
  __device__ __forceinline__ bool end(uint32_t bar, uint32_t parity) const {
    if (test_bar(bar, parity)) return true;
    for (int left = kEndTries; --left >= 0;)
      if (test_bar(bar, parity)) return true;
    fail();
    return false;
  }
  __device__ __forceinline__ void report(int* error) const {
    if (failed()) { *const_cast<volatile int*>(error) = 1; __threadfence_system(); }
  }
};
__device__ __forceinline__ void init_bar(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int N> __device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(on));
  return on;
}
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// NaN where one of them is
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// 2^x of a pair without the special function unit, which gives 16 results a cycle and is as busy as the tensor cores: x = n + f with n the
// nearest integer (found by adding 1.5 2^23), 2^f by the polynomial of degree 4 with the least relative error on [-1/2, 1/2] (2.6e-6, a
// hundredth of a 16-bit rounding; fitted by reweighted least squares), n added to its exponent.  Not below 2^-126.  A NaN, which an infinite logit
// becomes too, gives 2^128 (1 - 2^-24), infinite in 16 bits.
__device__ __forceinline__ float2 pow2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
  x.x = max_nan(x.x, -126.f); x.y = max_nan(x.y, -126.f);
  const float2 t = __fadd2_rn(x, magic), n = __fadd2_rn(t, minus), f = __fadd2_rn(x, make_float2(-n.x, -n.y));
  float2 p = make_float2(0.009570102207362652f, 0.009570102207362652f);
  p = __ffma2_rn(p, f, make_float2(0.05591786280274391f, 0.05591786280274391f));
  p = __ffma2_rn(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
  p = __ffma2_rn(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
  p = __ffma2_rn(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
  return make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + __float_as_uint(p.x)), __uint_as_float((__float_as_uint(t.y) << 23) + __float_as_uint(p.y)));
}
// 2^(a x + b) of sixteen values; POLY: half of them by the polynomial (8,192 rows, 9 heads, none / a quarter / half: d = 64 forward 245 / 241 /
// 237 us, dq 279 / 270 / 261; d = 128 dk and dv 457 / 445 / 436)
template <bool POLY> __device__ __forceinline__ void pow2_16(const uint32_t* x, float2 a, float2 b, float* y) {
#pragma unroll
  for (int e = 0; e < 16; e += 2) {
    const float2 z = __ffma2_rn(make_float2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), a, b);
    const float2 r = POLY && (e & 3) == 2 ? pow2_poly(z) : make_float2(pow2(z.x), pow2(z.y));
    y[e] = r.x; y[e + 1] = r.y;
  }
}

// ---- matrix instructions ----
// Geometry of operand tiles.  TERMS = 1: 16-bit values, sub-tiles of 64 values (128-byte rows and swizzle), one for DW = 64, two for 128.  TERMS = 3: float32
// values split into three bfloat16 terms, x = t0 + t1 + t2 to 2^-24, a sub-tile per term of DW = 32 or 64 values (64- or 128-byte rows and
// swizzle).  A product of two such operands takes the six products of terms that are above 2^-24 of it, small ones first.
template <int TERMS, int DW> struct Geometry {
  static constexpr int kRow = TERMS == 1 ? 128 : 2 * DW;      // bytes of a row
  static constexpr uint32_t kSub = kTile * kRow;              // bytes of a sub-tile
  static constexpr int kSubs = TERMS == 1 ? DW / 64 : 3;
  // Tiles that stream through: a ring, the two kinds of tile in turn; tile j sits in slot j % R.
  static constexpr int kRing = TERMS == 1 ? (DW == 128 ? 4 : 8) : DW == 32 ? 6 : 2;
  // a ring of one tile of each kind: the reverse kernels make the next logits only behind the product that reads the tile in its slot
  static constexpr bool kShort = TERMS == 3 && DW == 64;
  // Where tensor memory has room for P and dS beside the logits and dP they are made from, the next tile's logits are made as soon as these
  // have been read, and not behind the product that reads P: a product's way through barriers and back is longer than itself.
  static constexpr bool kEarly = TERMS == 1 && DW == 64, kEarlyDq = kEarly || (TERMS == 3 && DW == 32);
  // Descriptor: its low word holds the address, so that steps are additions to it; the high word is a constant.  K-major: 16 contracted values
  // are 32 bytes further, 64 are a sub-tile further; groups of eight rows lie 8 rows apart.  MN-major: 16 contracted rows are 16 rows
  // further, the next values of N a sub-tile.
  static constexpr uint32_t kHigh = (8 * kRow >> 4) | (1u << 14) | ((kRow == 128 ? 2u : 4u) << 29);
  static __device__ __forceinline__ uint32_t low(uint32_t addr, bool mn_major) { return ((addr >> 4) & 0x3FFF) | ((mn_major ? kSub >> 4 : 1) << 16); }
  static constexpr uint32_t step_k(int k) { return ((k & 3) * 32 + (k >> 2) * kSub) >> 4; }
  static constexpr uint32_t kStepMn = 16 * kRow >> 4, kStepTerm = kSub >> 4;
};
template <typename T> __device__ __forceinline__ uint32_t idesc(int n, bool b_mn_major) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// The whole warp runs the issue code, the elected lane (`on`) issues: descriptors stay in uniform registers.  All loops around these are
// unrolled: with addresses formed between two instructions a thread got one out every 120 to 170 cycles, twice what it takes to run.
template <uint32_t HIGH> __device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 x, {%1, %6};\n\tmov.b64 y, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "r"(on), "n"(HIGH) : "memory");
}
template <uint32_t HIGH> __device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 y, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n" ::"r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "r"(on), "n"(HIGH) : "memory");
}
__device__ __forceinline__ void commit(uint32_t on, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar), "r"(on) : "memory");
}
// D[128 x 128] = A B^T over d columns, both tiles in shared memory
template <typename T, int TERMS, int DW> __device__ __forceinline__ void product_rows(uint32_t on, uint32_t dst, uint32_t a, uint32_t b, int d) {
  using G = Geometry<TERMS, DW>;
  const uint32_t la = G::low(a, false), lb = G::low(b, false), id = idesc<T>(kTile, false);
  if constexpr (TERMS == 1) {
    const int steps = d / 16;
#pragma unroll
    for (int k = 0; k < DW / 16; ++k)
      if (k < steps) mma_ss<G::kHigh>(on, dst, la + G::step_k(k), lb + G::step_k(k), id, k > 0);
  } else {
#pragma unroll
    for (int e = 0; e < 6; ++e) {
      // (2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)
      const uint32_t x = e == 0 ? 2 : (e == 2 || e == 3), y = e == 1 ? 2 : (e == 2 || e == 4);
#pragma unroll
      for (int k = 0; k < DW / 16; ++k) mma_ss<G::kHigh>(on, dst, la + x * G::kStepTerm + G::step_k(k), lb + y * G::kStepTerm + G::step_k(k), id, (e | k) > 0);
    }
  }
}
// where a 128 x 128 operand packed to 16 bits sits in tensor memory: 64 columns in two halves `gap` columns apart, for each of its terms
struct Packed { uint32_t at[3]; int gap[3]; };
// D[128 x d] (+)= A B: A in tensor memory, B a tile with its rows contracted.  Three terms and DW = 32: two terms of B side by side as N = 64,
// D = [.. t0 | .. t1 and t2], whose halves are to be added; started afresh every time.
// FIRST, LAST: 16ths of the contracted index, [0, 8) for all.
template <typename T, int TERMS, int DW, int FIRST = 0, int LAST = 8>
__device__ __forceinline__ void product_cols(uint32_t on, uint32_t dst, const Packed a, uint32_t b, int d, uint32_t acc) {
  using G = Geometry<TERMS, DW>;
  static_assert(TERMS == 1 || LAST - FIRST == 8, "three terms take the whole index at once");
  const uint32_t lb = G::low(b, true);
  auto steps = [&](int term, uint32_t bt, uint32_t to, int n, uint32_t add) {
    const uint32_t id = idesc<T>(n, true);
#pragma unroll
    for (int k = FIRST; k < LAST; ++k) mma_ts<G::kHigh>(on, to, a.at[term] + (k & 3) * 8 + (k >> 2) * a.gap[term], bt + k * G::kStepMn, id, add | (k > 0));
  };
  if constexpr (TERMS == 1) {
    steps(0, lb, dst, d, acc);
  } else if constexpr (DW == 32) {
    steps(2, lb, dst, 32, 0);
    steps(0, lb + 2 * G::kStepTerm, dst + 32, 32, 0);
    steps(1, lb, dst, 64, 1);
    steps(0, lb, dst, 64, 1);
  } else {
    steps(2, lb, dst, 64, 0);
    steps(0, lb + 2 * G::kStepTerm, dst, 64, 1);
    steps(1, lb + G::kStepTerm, dst, 64, 1);
    steps(1, lb, dst, 64, 1);
    steps(0, lb + G::kStepTerm, dst, 64, 1);
    steps(0, lb, dst, 64, 1);
  }
}

// ---- tensor memory ----
#define R8(x, o) x[o], x[o + 1], x[o + 2], x[o + 3], x[o + 4], x[o + 5], x[o + 6], x[o + 7]
#define O8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define I8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : O8(r, 0), O8(r, 8), O8(r, 16), O8(r, 24) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : O8(r, 0), O8(r, 8) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(addr), I8(r, 0), I8(r, 8) : "memory");
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), I8(r, 0) : "memory");
}
#undef R8
#undef O8
#undef I8
// waits for the loads of N registers; what reads them stays behind the wait
template <int N> __device__ __forceinline__ void wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// sixteen values as eight packed pairs, in one or three terms, to the places of `to` that belong to column `c` (a multiple of 16 of the
// 64 of a half, or of all 128 where the halves lie together)
template <typename T, int TERMS> __device__ __forceinline__ void put16(const Packed& to, uint32_t lanes, int c, const float* v) {
  uint32_t p[8];
  float r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = v[i];
#pragma unroll
  for (int term = 0; term < TERMS; ++term) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = packed::Half<T>::pack(r[2 * i], r[2 * i + 1]);
      if (term + 1 < TERMS) {
        const float2 u = packed::Half<T>::unpack(p[i]);
        r[2 * i] -= u.x; r[2 * i + 1] -= u.y;
      }
    }
    st8(lanes + to.at[term] + c / 2, p);
  }
}

// ---- loading ----
struct Maps { CUtensorMap q, k, v, g; };
__device__ __forceinline__ void tma(uint32_t dst, const CUtensorMap* map, int x, int row, int head, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(head), "r"(bar) : "memory");
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// The whole loading warp calls it.  rows: how many of the tile's 128 rows belong to the structure; where `clear`, the others are cleared
// (through `fix`, a barrier of this warp's own, and its parity).  Behind a failure nothing is issued any more: a slot may have been given back by
// products that did not wait for its tile, and its copy may still be under way.
template <int TERMS, int DW> struct Loader {
  static constexpr uint32_t kSub = Geometry<TERMS, DW>::kSub;
  static constexpr int subs = Geometry<TERMS, DW>::kSubs;
  int lane;
  uint32_t fix;
  Wait wait;
  uint32_t parity = 0;
  bool ok = true;            // no wait has run out
  __device__ __forceinline__ void need(uint32_t bar, uint32_t phase) { ok = wait.of_loader(bar, phase) && !wait.failed() && ok; }
  __device__ __forceinline__ bool go() const { return lane == 0 && ok; }      // whether this lane issues
  __device__ __forceinline__ void copies(uint32_t dst, const CUtensorMap* map, int row, int head, uint32_t bar) const {
    for (int x = 0; x < subs; ++x) tma(dst + x * kSub, map, TERMS == 1 ? 64 * x : 0, row, TERMS == 1 ? head : 3 * head + x, bar);
  }
  // returns 1 in the first lane where the tile was handed over or is on its way
  __device__ __forceinline__ int tile(uint32_t dst, const CUtensorMap* map, int row, int head, uint32_t full, int rows, bool clear) {
    const bool issue = go();
    if (!clear || rows >= kTile) {
      if (issue) { expect(full, subs * kSub); copies(dst, map, row, head, full); }
      __syncwarp();
      return issue;
    }
    if (issue) { expect(fix, subs * kSub); copies(dst, map, row, head, fix); }
    __syncwarp();
    need(fix, parity);
    if (issue && !ok) wait.end(fix, parity);
    parity ^= 1;
    for (int x = 0; x < subs; ++x)
      for (int b = rows * Geometry<TERMS, DW>::kRow + lane * 16; b < (int)kSub; b += 512)
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + x * kSub + b), "r"(0) : "memory");
    fence_smem();
    __syncwarp();
    if (issue && ok) arrive(full);
    __syncwarp();
    return issue && ok;
  }
};

__device__ __forceinline__ void alloc_tmem(uint32_t* where, int columns = 512) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(where)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void free_tmem(uint32_t tmem, int columns = 512) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

}  // namespace tc
}  // namespace so3lr
