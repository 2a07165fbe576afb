// Attention inside the structures of a packed batch on the tensor cores (tcgen05): forward and the two halves of the reverse pass, for
// structures long enough to fill tiles of 128 rows.  The mathematics is that of packed_mma.cuh.  16-bit operands as they are; float32 with up to 64
// values a head as three bfloat16 terms each (Geometry), with accumulators over the walked side in registers, because the tensor cores cut
// what they add to an accumulator (2^-24 of the sum a step).
//
// A CTA has the SM to itself (a forward one of one tile: half of it): eight warps do the softmax (a thread per row, or per row and half of the
// columns), one warp issues the matrix instructions, one loads tiles, two fetch the statistics that dk and dv need.  Accumulators and P /
// dS live in tensor memory: P and dS go back there packed to 16 bits, and are the A operand of the next product, so shared memory
// carries q, k, v and g only.
//
// Bound by the tensor cores beside the elementwise work of eight warps.  8,192 rows, 9 heads x 128 bfloat16: forward 261 us (1.18 PFLOP/s), dq 382 (1.21),
// dk and dv 444 (1.39; cuBLAS 1.67), the tensor cores busy 61, 59 and 73 % of the time and the schedulers 40 to 53 %.  With 64 values a head
// a tile has half of the products, each of them no shorter for its 64 columns, and the same elementwise work (237, 297, 351 us; tensor 31, 37,
// 42 % busy, schedulers 49 to 56 %): what is left is the latency of two warps per scheduler.  float32, 9 x 32: 425, 517, 796 us, tensor 55 to 66 %.
// The two reverse kernels form seven products where one with atomic sums would form five; they give the same bits every time.
#include "packed_tc.cuh"

#include <algorithm>
#include <mutex>

namespace so3lr {

namespace {

using namespace tc;

// barriers and scratch behind the tiles
constexpr int kBars = 40;
// What a CTA works on at a time: a tile of rows from row0 on of one head (or key head) h against n tiles of the other side, a
// piece of an item's walk.  n < 0: there is no more.
struct Job {
  int q0, lq, c0, lk, h, row0, n, piece;
  int k0;               // forward, dq: first key
  int n0, n1;           // forward: tiles of keys that the two tiles of rows meet (n is the larger count)
  int i0, per, j0;      // dk and dv: first query; tiles of queries of a head from there on; the job's first one among those of all heads of the group
  float size_v;         // dq of float16: the largest |v|
  int shift;            // dk and dv of float16: the power of two of dS (grad_shift)
};
struct Tail {
  unsigned long long bars[kBars];
  uint32_t tmem;
  int failed;
  Job jobs[2];       // the jobs at hand
  int tiles[2];      // reverse kernels: tiles of those that have any, 0 behind the last one
};
template <typename T, int TERMS> struct Operand { using type = T; };
template <> struct Operand<float, 3> { using type = __nv_bfloat16; };
// 16 values to a row of the result
template <typename T> __device__ __forceinline__ void store16(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    uint32_t u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = packed::Half<T>::pack(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
    *reinterpret_cast<uint4*>(p + 8) = make_uint4(u[4], u[5], u[6], u[7]);
  } else {
#pragma unroll
    for (int e = 0; e < 16; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
  }
}
// adds W columns of a tile's fresh product to registers; DW = 32: of both halves of D (see product_cols)
template <int DW, int W> __device__ __forceinline__ void add_cols(uint32_t at, float* o) {
#pragma unroll
  for (int c = 0; c < W; c += 16) {
    uint32_t x[16];
    ld16(at + c, x);
    wait_ld(x);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[c + e] += __uint_as_float(x[e]);
    if (DW == 32) {
      ld16(at + 32 + c, x);
      wait_ld(x);
#pragma unroll
      for (int e = 0; e < 16; ++e) o[c + e] += __uint_as_float(x[e]);
    }
  }
}
// sub-tiles need 1024-byte alignment
__device__ __forceinline__ unsigned char* aligned_smem(unsigned char* p) { return p + ((1024u - (smem_addr(p) & 1023u)) & 1023u); }

// ---- jobs -----------------------------------------------------------------------------------------------------------
// A CTA stays on its SM and works through jobs, so that a job's first tiles come in and its first products run while the last results of the
// one before leave: with a CTA per job its start and end took 5 to 6 us, now 2 to 3.  dq / dk and dv, a CTA per job -> this, us: 24 structures of 150 to
// 900 rows, 16 heads x 64, 124 / 147 -> 100 / 121; 64 of 64 to 128, 8 x 128, 28 / 32 -> 20 / 26; 8 causal ones of 2,000, 40 x 128, 613 / 588 ->
// 520 / 592; one of 8,192, 9 x 64, 290 / 351 -> 297 / 351 (a job of 64 tiles has no start to hide).  The loading warp takes jobs from a queue, the
// longest first, and passes them on through shared memory (equal shares instead: SMs differ in their pace by up to 15 %; 5,000 rows, 4 x 32
// float32, dk and dv 187 us with the queue, 219 without).
// Jobs are passed on after a failure too, so that the rows of all of them are written; false where that is at an end as well.
__device__ __forceinline__ bool publish_job(Tail* tail, int m, const Job& j, uint32_t full, uint32_t free, int lane, const Wait& wait) {
  if (m >= 2 && !__all_sync(0xffffffffu, wait.end(free + 8 * (m & 1), ((m >> 1) - 1) & 1))) return false;
  if (lane == 0) { tail->jobs[m & 1] = j; arrive(full + 8 * (m & 1)); }
  __syncwarp();
  return true;
}
// a warp's m-th job
__device__ __forceinline__ Job take_job(const Tail* tail, int m, uint32_t full, uint32_t free, int lane, const Wait& wait) {
  const bool ok = wait.end(full + 8 * (m & 1), (m >> 1) & 1);
  Job j = tail->jobs[m & 1];
  if (!__all_sync(0xffffffffu, ok)) j.n = -1;
  if (lane == 0) arrive(free + 8 * (m & 1));
  return j;
}
// the next job's index
__device__ __forceinline__ int next_index(int* queue, int at, int last, int lane) {
  int index = 0;
  if (lane == 0) index = queue ? at + atomicAdd(queue, 1) : last;
  return __shfl_sync(0xffffffffu, index, 0);
}

// ---- forward --------------------------------------------------------------------------------------------------------
// 256 queries of one head: two tiles of 128 rows take turns, so that the exponentials of one run beside the products of the other.
// Tensor memory: logits of tile t at 128 t, its output at 256 + 128 t, one tile's at 128; P of a tile replaces its logits.  (Up to 64 values a head,
// one tile: logits at 0, output at 128, P at 192.  float32: logits at 256 t, the three terms of P from there on, its output at 256 t + 192.)
// The running maximum that the exponentials refer to is raised only where it would grow by more than kLag (in log2): P stays below
// 2^(kHead + kLag), and the output, which the tensor cores add to, is rescaled a few times per row instead of once per tile of keys.
enum FwdBar { kFull, kEmpty = kFull + 8, kQFull = kEmpty + 8, kQFree = kQFull + 2, kSFull = kQFree + 2, kPFull = kSFull + 2 /* tile + 2 half */, kOFull = kPFull + 4,
              kFix = kOFull + 2, kDone, kSRead, kJob = kSRead + 2, kJobFree = kJob + 2, kFwdBars = kJobFree + 2 };
template <int TILES> __device__ __forceinline__ Job forward_job(const PackedArgs& a, int index) {
  Job j = {};
  j.n = -1;
  if (index >= a.jobs) return j;
  const int unit = index / a.pieces;
  const int4 item = __ldg(a.items + unit / a.hq);
  j.piece = index % a.pieces; j.h = unit % a.hq;
  j.q0 = __ldg(a.start_q + item.x); j.lq = __ldg(a.start_q + item.x + 1) - j.q0; j.c0 = __ldg(a.start_kv + item.x); j.lk = __ldg(a.start_kv + item.x + 1) - j.c0;
  j.row0 = item.y * TILES * kTile;
  // keys that a tile of rows meets: [0, end), and tiles of keys
  const int end1 = item.w, end0 = TILES == 2 && a.causal ? min(end1, max(0, min(j.lq, j.row0 + kTile) + j.lk - j.lq)) : end1;
  const int all0 = (end0 + kTile - 1) / kTile, all1 = TILES == 2 && j.row0 + kTile < j.lq ? (end1 + kTile - 1) / kTile : 0;
  const int all = max(all0, all1), share = all / a.pieces, more = all % a.pieces, first = j.piece * share + min(j.piece, more);
  j.n = share + (j.piece < more); j.k0 = first * kTile;
  j.n0 = min(j.n, max(0, all0 - first)); j.n1 = min(j.n, max(0, all1 - first));
  return j;
}

// TILES = 1: a CTA has one tile and half of an SM, which two of them share: one's start and end pass beside the other's work.
template <int TERMS, int DW, int TILES> struct Forward {
  static constexpr int kMma = 4 * TILES, kLoad = kMma + 1, kThreads = 128 * TILES + 128;
  // registers: 256 x 208 + 128 x 88 = 384 x 168; 128 x 200 + 128 x 56 = 256 x 128
  static constexpr int kRegs = TILES == 2 ? 208 : 200, kOtherRegs = TILES == 2 ? 88 : 56;
  static constexpr int kRing = TILES == 2 ? Geometry<TERMS, DW>::kRing : TERMS == 3 ? 3 : DW == 128 ? 2 : 4;
  static constexpr int kSmem = 1024 + (TILES + kRing) * Geometry<TERMS, DW>::kSubs * (int)Geometry<TERMS, DW>::kSub + (int)sizeof(Tail);
  static_assert(TILES == 2 || kSmem <= 232448 / 2, "two CTAs on an SM");
  // Whether CTAs take jobs from a queue, or have one each.  us, one / queue: 8 causal prompts of 2,000, 40 heads x 128, 509 / 452; 24 structures of 150 to
  // 900, 16 x 64, 104 / 96; one of 8,192, 9 x 128 260 / 261, 9 x 64 234 / 237; but float32, whose registers spill over what a job takes, 32 of 256,
  // 4 x 32, 15.1 / 16.8, one of 5,000 101 / 113, one of 8,192, 9 x 32, 425 / 486.
  static constexpr bool kQueued = TERMS == 1;
};
template <typename T, int TERMS, int DW, int TILES>
__global__ void __launch_bounds__(Forward<TERMS, DW, TILES>::kThreads, TILES == 2 ? 1 : 2) forward_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  using M = typename Operand<T, TERMS>::type;
  using G = Geometry<TERMS, DW>;
  using F = Forward<TERMS, DW, TILES>;
  constexpr int kMmaWarp = F::kMma, kLoadWarp = F::kLoad;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d;
  constexpr int tile_bytes = G::kSubs * (int)G::kSub, R = F::kRing;
  Tail* tail = reinterpret_cast<Tail*>(smem + (TILES + R) * tile_bytes);
  const uint32_t sq = smem_addr(smem), ring = sq + TILES * tile_bytes, bar0 = smem_addr(tail->bars);
  const Wait wait{smem_addr(&tail->failed), a.wait_tries};
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem, 256 * TILES);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kFwdBars; ++i) init_bar(bar(i), (i >= kPFull && i < kPFull + 4) || (i >= kSRead && i < kSRead + 2) ? kTile : i >= kJobFree ? 4 * TILES + 1 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;
  // columns from one tile's logits to the other's, output of a tile, columns from one output to the other, P
  constexpr uint32_t kStride = TERMS == 1 ? kTile : 256, kOut = TERMS == 1 ? kTile * TILES : 192, kOutStride = TERMS == 1 ? DW : 256;
  static_assert(!G::kEarly || TILES == 1, "P beside the logits: room for one tile's");
  auto p_at = [](int t) { return G::kEarly ? kOut + 64 : kStride * t; };

  auto job_at = [&](int m) {
    if constexpr (F::kQueued) return take_job(tail, m, bar(kJob), bar(kJobFree), lane, wait);
    else return forward_job<TILES>(a, blockIdx.x);
  };

  if (warp >= kMmaWarp) {
    fewer_regs<F::kOtherRegs>();
    if (warp == kMmaWarp) {
      const uint32_t on = elect_one();
      auto need = [&](uint32_t b, uint32_t parity) { wait(b, parity); fence_after(); };
      // tiles are counted over all jobs: keys are tiles 0, 2, .. of the ring, values 1, 3, ..; g: the tile at hand, base: tiles of the two tiles of rows
      // before the job
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };
      auto ready = [&](int j) { need(bar(kFull + j % R), (j / R) & 1); };
      auto give = [&](int j) { commit(on, bar(kEmpty + j % R)); };
      int g = 0, base[2] = {0, 0}, jobs_of[2] = {0, 0};
      for (int m = 0; F::kQueued || m < 1; ++m) {
        const Job j = job_at(m);
        const int n = __shfl_sync(0xffffffffu, j.n, 0), n0 = __shfl_sync(0xffffffffu, j.n0, 0), n1 = __shfl_sync(0xffffffffu, j.n1, 0);
        if (n < 0) break;
        if (n == 0) continue;
        ready(2 * g);
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const int nt = t ? n1 : n0;
          if (nt == 0) continue;
          need(bar(kQFull + t), jobs_of[t] & 1);
          ++jobs_of[t];
          product_rows<M, TERMS, DW>(on, tmem + kStride * t, sq + t * tile_bytes, slot(2 * g), d);
          commit(on, bar(kSFull + t));
          if (nt == 1) commit(on, bar(kQFree + t));
        }
        give(2 * g);
        for (int i = 0; i < n; ++i, ++g) {
          auto logits = [&](int t) {
            const int nt = t ? n1 : n0;
            if (i + 1 >= nt) return;
            product_rows<M, TERMS, DW>(on, tmem + kStride * t, sq + t * tile_bytes, slot(2 * g + 2), d);
            commit(on, bar(kSFull + t));
            if (i + 2 == nt) commit(on, bar(kQFree + t));
          };
          if (i + 1 < n) ready(2 * g + 2);
          if (G::kEarly) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
              if (i + 1 >= (t ? n1 : n0)) continue;
              need(bar(kSRead + t), (base[t] + i) & 1);
              logits(t);
            }
            if (i + 1 < n) give(2 * g + 2);
          }
          ready(2 * g + 1);
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            const int nt = t ? n1 : n0;
            if (i >= nt) continue;
            need(bar(kPFull + t), (base[t] + i) & 1);
            const uint32_t at = tmem + p_at(t), out = tmem + kOut + kOutStride * t;
            const Packed p{{at, at + 64, at + 128}, {32, 32, 32}};
            if constexpr (TERMS == 1) {      // the first half of the keys while the exponentials of the second are formed
              product_cols<M, TERMS, DW, 0, 4>(on, out, p, slot(2 * g + 1), d, i > 0);
              need(bar(kPFull + 2 + t), (base[t] + i) & 1);
              product_cols<M, TERMS, DW, 4, 8>(on, out, p, slot(2 * g + 1), d, 1);
            } else {
              product_cols<M, TERMS, DW>(on, out, p, slot(2 * g + 1), d, 0);
            }
            if (!G::kEarly) logits(t);
            if (G::kEarly || i + 1 == nt) commit(on, bar(kOFull + t));
          }
          give(2 * g + 1);
          if (!G::kEarly && i + 1 < n) give(2 * g + 2);
        }
        base[0] += n0; base[1] += n1;
      }
      commit(on, bar(kDone));      // no matrix instruction is under way when the CTA ends
      wait.end(bar(kDone), 0);
    } else if (warp == kLoadWarp) {
      Loader<TERMS, DW> ld{lane, bar(kFix), wait};
      int g = 0, issued = 0, jobs_of[2] = {0, 0}, issued_of[2] = {0, 0};      // tiles; those whose copies the first lane has issued
      bool stop = false;          // after a failure: jobs without any tile
      for (int m = 0, index = blockIdx.x; F::kQueued || m < 1; ++m) {
        Job j = forward_job<TILES>(a, index);
        if (stop) { j.n = min(j.n, 0); j.n0 = j.n1 = 0; }
        const int kvh = j.h / a.group;
        if constexpr (F::kQueued) { if (!publish_job(tail, m, j, bar(kJob), bar(kJobFree), lane, wait)) break; }
        if (j.n < 0) break;
        for (int i = 0; i < 2 * j.n; ++i, ++g) {
          if (i == 1) {      // behind the first tile of keys, which finds room earlier
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
              if ((t ? j.n1 : j.n0) == 0) continue;
              if (jobs_of[t] > 0) ld.need(bar(kQFree + t), (jobs_of[t] - 1) & 1);
              ++jobs_of[t];
              issued_of[t] += ld.tile(sq + t * tile_bytes, &maps.q, j.q0 + j.row0 + t * kTile, j.h, bar(kQFull + t), kTile, false);
            }
          }
          if (g >= R) ld.need(bar(kEmpty + g % R), (g / R - 1) & 1);
          const int r = j.k0 + (i >> 1) * kTile;
          issued += ld.tile(ring + (g % R) * tile_bytes, (i & 1) ? &maps.v : &maps.k, j.c0 + r, kvh, bar(kFull + g % R), j.lk - r, i & 1);
        }
        if (F::kQueued) { index = next_index(a.queue, gridDim.x, a.jobs, lane); stop = __any_sync(0xffffffffu, wait.failed()); }
      }
      // no copy is under way when the CTA ends
      for (int t = max(0, issued - R); t < issued; ++t) wait.end(bar(kFull + t % R), (t / R) & 1);
#pragma unroll
      for (int t = 0; t < TILES; ++t) if (issued_of[t] > 0) wait.end(bar(kQFull + t), (issued_of[t] - 1) & 1);
      __syncwarp();
    }
  } else {
    more_regs<F::kRegs>();
    const int t = warp >> 2, w = warp & 3;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w) << 16), ts = lanes + kStride * t, to = lanes + kOut + kOutStride * t;
    constexpr int kOwn = TERMS == 1 ? 1 : DW;
    constexpr float head = kHead<T, true>;
    int g = 0, job = 0;                        // tiles, and jobs that had any
    Job j = job_at(0);
    for (int k = 1; j.n >= 0; ++k) {
      const int nt = t ? j.n1 : j.n0, off = j.lk - j.lq, row = j.row0 + t * kTile + w * 32 + lane, first = j.row0 + t * kTile + w * 32;
      float own[kOwn];                         // the output so far (float32)
#pragma unroll
      for (int c = 0; c < kOwn; ++c) own[c] = 0.f;
      // last key that this row sees, and that the warp's first row sees
      const int lim = min(a.causal ? row + off : j.lk - 1, j.lk - 1), lim_first = min(a.causal ? first + off : j.lk - 1, j.lk - 1);
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < nt; ++i, ++g) {
        wait(bar(kSFull + t), g & 1);
        fence_after();
        if constexpr (TERMS == 3) { if (i > 0) add_cols<DW, DW>(to, own); }
        uint32_t x[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) ld32(ts + c, x + c);
        wait_ld(x);
        if (G::kEarly) { fence_before(); arrive(bar(kSRead + t)); }
        const int kb = j.k0 + i * kTile;
        const bool masked = kb + kTile - 1 > lim_first;
        if (masked) {
#pragma unroll
          for (int c = 0; c < kTile; ++c) if (kb + c > lim) x[c] = 0xff800000u;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kTile; c += 8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1]));
        }
        const float mn = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * a.scale_log2);
        const bool raise = mn > m + kLag<T>;      // true where there was none yet
        if (G::kEarly && i > 0) { wait(bar(kOFull + t), (g - 1) & 1); fence_after(); }      // the output and P are free
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? pow2(m - mn) : 1.f;
          if (raise) m = mn;
          l *= f;
          if constexpr (TERMS == 3) {
#pragma unroll
            for (int c = 0; c < kOwn; ++c) own[c] *= f;
          } else if (i > 0) {
            for (int c = 0; c < d; c += 16) {
              uint32_t o[16];
              ld16(to + c, o);
              wait_ld(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              st16(to + c, o);
            }
          }
        }
        const float u = m == -INFINITY ? 0.f : head - m;
        float2 sums[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[e] = make_float2(0.f, 0.f);
        const Packed at{{p_at(t), p_at(t) + 64, p_at(t) + 128}, {}};
        const float2 scale = make_float2(a.scale_log2, a.scale_log2), ref = make_float2(u, u);
#pragma unroll
        for (int c = 0; c < kTile; c += 32) {
          float y[32];
          // a masked logit has to give zero, which the polynomial does not
          if (TERMS == 1 && !masked) { pow2_16<true>(x + c, scale, ref, y); pow2_16<true>(x + c + 16, scale, ref, y + 16); }
          else { pow2_16<false>(x + c, scale, ref, y); pow2_16<false>(x + c + 16, scale, ref, y + 16); }
#pragma unroll
          for (int e = 0; e < 32; e += 2) sums[(e >> 1) & 3] = __fadd2_rn(sums[(e >> 1) & 3], make_float2(y[e], y[e + 1]));
          put16<M, TERMS>(at, lanes, c, y);
          put16<M, TERMS>(at, lanes, c + 16, y + 16);
          if (TERMS == 1 && c == kTile / 2 - 32) {
            wait_st();
            fence_before();
            arrive(bar(kPFull + t));
          }
        }
        const float2 sum = __fadd2_rn(__fadd2_rn(sums[0], sums[1]), __fadd2_rn(sums[2], sums[3]));
        l += sum.x + sum.y;
        wait_st();
        fence_before();
        arrive(bar(kPFull + t + (TERMS == 1 ? 2 : 0)));
      }
      if (nt > 0) {
        wait(bar(kOFull + t), (G::kEarly ? g - 1 : job) & 1);
        ++job;
        fence_after();
      }
      if constexpr (TERMS == 3) { if (nt > 0) add_cols<DW, DW>(to, own); }
      const bool there = row < j.lq, bad = wait.failed();
      if (a.pieces > 1) {      // the share: o as it is, with its maximum and sum
        const long long slot = ((long long)j.piece * a.hq + j.h) * a.nq + j.q0 + row;
        if (there) a.part_ml[slot] = make_float2(m - head, bad ? NAN : l);
        float* dst = a.part_o + slot * d;
        if (nt > 0) {
          if constexpr (TERMS == 3) {
#pragma unroll
            for (int c = 0; c < DW; c += 16) if (there && c < d) store16(dst + c, own + c);
          } else {
            for (int c = 0; c < d; c += 16) {
              uint32_t o[16];
              float y[16];
              ld16(to + c, o);
              wait_ld(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(o[e]);
              if (there) store16(dst + c, y);
            }
          }
        }
      } else {
        const float inv = bad ? NAN : l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        const long long at = ((long long)(j.q0 + row) * a.hq + j.h) * d;
        T *dst = static_cast<T*>(a.out) + at, *rest = a.out_rest ? static_cast<T*>(a.out_rest) + at : nullptr;
        if constexpr (TERMS == 3) {
#pragma unroll
          for (int c = 0; c < kOwn; ++c) own[c] *= inv;
#pragma unroll
          for (int c = 0; c < DW; c += 16) if (there && c < d) store16(dst + c, own + c);
        } else {
          for (int c = 0; c < d; c += 16) {
            uint32_t o[16];
            float y[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0;
            if (nt > 0) { ld16(to + c, o); wait_ld(o); }
#pragma unroll
            for (int e = 0; e < 16; ++e) y[e] = __uint_as_float(o[e]) * inv;
            if (there) {
              store16(dst + c, y);
              if (rest) {
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                  const float2 r = packed::Half<T>::unpack(packed::Half<T>::pack(y[e], y[e + 1]));
                  y[e] -= r.x; y[e + 1] -= r.y;
                }
                store16(rest + c, y);
              }
            }
          }
        }
        if (there && a.lse) a.lse[(long long)j.h * a.nq + j.q0 + row] = bad ? NAN : l == 0.f ? -INFINITY : m - head + log2f(l);
      }
      if constexpr (!F::kQueued) break;
      j = job_at(k);
    }
    fence_before();
  }
  __syncthreads();
  if (tid == 0) wait.report(a.error);
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem, 256 * TILES); }
}

// ---- reverse: dq ----------------------------------------------------------------------------------------------------
// dq: 128 queries of one head.  Tensor memory: logits at 0, dP at 128 (dS replaces it, in two halves), dq at 256 (float32: the third term of dS
// at 256, dq at 320; where there is room dS at 256 and dq behind it).  The two groups of four warps have 64 columns each of every row.  The
// next tile's logits are made as soon as these have been read, so that its exponentials run beside the products dS k and g v^T.
enum DqBar { kdqFull, kdqEmpty = kdqFull + 8, kdqQ = kdqEmpty + 8, kdqQFree, kdqS, kdqSRead, kdqDp, kdqDpRead, kdqDs, kdqDsDone, kdqOut, kdqFix, kdqDone, kdqJob,
             kdqJobFree = kdqJob + 2, kDqBars = kdqJobFree + 2 };
__device__ __forceinline__ Job dq_job(const PackedArgs& a, int index) {
  Job j = {};
  j.n = -1;
  if (index >= a.jobs) return j;
  const int unit = index / a.pieces;
  const int4 item = __ldg(a.items + unit / a.hq);
  j.piece = index % a.pieces; j.h = unit % a.hq;
  j.q0 = __ldg(a.start_q + item.x); j.lq = __ldg(a.start_q + item.x + 1) - j.q0; j.c0 = __ldg(a.start_kv + item.x); j.lk = __ldg(a.start_kv + item.x + 1) - j.c0;
  j.row0 = item.y * kTile;
  if (a.largest) j.size_v = __uint_as_float(__ldg(a.largest + ((long long)item.x * a.hk + j.h / a.group) * 2 + 1));
  const int all = (item.w + kTile - 1) / kTile, share = all / a.pieces, more = all % a.pieces;
  j.k0 = (j.piece * share + min(j.piece, more)) * kTile; j.n = share + (j.piece < more);
  return j;
}

template <typename T, int TERMS, int DW>
__global__ void __launch_bounds__(kThreads, 1) dq_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  using M = typename Operand<T, TERMS>::type;
  using G = Geometry<TERMS, DW>;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d;
  constexpr int tile_bytes = G::kSubs * (int)G::kSub, R = G::kRing;
  Tail* tail = reinterpret_cast<Tail*>(smem + (2 + R) * tile_bytes);
  const uint32_t sq = smem_addr(smem), sg = sq + tile_bytes, ring = sg + tile_bytes, bar0 = smem_addr(tail->bars);
  const Wait wait{smem_addr(&tail->failed), a.wait_tries};
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kDqBars; ++i) init_bar(bar(i), i == kdqSRead || i == kdqDpRead || i == kdqDs ? 256 : i >= kdqJobFree ? 8 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;
  constexpr bool E = G::kEarlyDq;
  constexpr uint32_t kDs = E ? 256 : kTile, kOut = E ? (TERMS == 1 ? 320 : 448) : (TERMS == 1 ? 256 : 320);

  // Tiles are counted over all jobs (keys are tiles 0, 2, .. of the ring, values 1, 3, ..), and so are jobs that have any: barriers turn with these.
  if (warp >= kMmaWarp) {
    fewer_regs<kOtherRegs>();
    if (warp == kMmaWarp) {
      const uint32_t on = elect_one();
      auto need = [&](uint32_t b, uint32_t parity) { wait(b, parity); fence_after(); };
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };
      auto ready = [&](int j) { need(bar(kdqFull + j % R), (j / R) & 1); };
      auto give = [&](int j) { commit(on, bar(kdqEmpty + j % R)); };
      // Logits and dP run a tile ahead: tile g + 1 of all, tile i + 1 of the job's n.  The loop is as short as it can be (the loading warp says how
      // many tiles a job has, every product stands in one place, so that a job starts a step early): what this warp does between two
      // instructions keeps the tensor cores waiting.  It waits for a job only behind the last product of the one before, without which the
      // compute warps do not get to the jobs in between that have no tiles.
      int g = -1;
      for (int job = 0;; ++job) {
        need(bar(kdqQ), job & 1);
        const int n = __shfl_sync(0xffffffffu, wait.failed() ? 0 : tail->tiles[job & 1], 0);
        if (n == 0) break;
        for (int i = -1; i < n; ++i) {
          const bool more = i + 1 < n;
          auto logits = [&] {
            if (!more) return;
            ready(2 * g + 2);
            if (g >= 0) need(bar(kdqSRead), g & 1);
            product_rows<M, TERMS, DW>(on, tmem, sq, slot(2 * g + 2), d);
            commit(on, bar(kdqS));
          };
          auto dp = [&] {
            if (!more) return;
            ready(2 * g + 3);
            if (E && g >= 0) need(bar(kdqDpRead), g & 1);
            product_rows<M, TERMS, DW>(on, tmem + kTile, sg, slot(2 * g + 3), d);
            commit(on, bar(kdqDp));
            give(2 * g + 3);
            if (i + 2 == n) commit(on, bar(kdqQFree));
          };
          if (!G::kShort) logits();
          if (E) dp();
          if (i >= 0) {
            need(bar(kdqDs), g & 1);
            const uint32_t at = tmem + kDs;
            product_cols<M, TERMS, DW>(on, tmem + kOut, E ? Packed{{at, at + 64, at + 128}, {32, 32, 32}} : Packed{{at, at + 32, tmem + 256}, {64, 64, 32}},
                                       slot(2 * g), d, i > 0);
            if (E) commit(on, bar(kdqDsDone));
            if (!more) commit(on, bar(kdqOut));
            give(2 * g);
          }
          if (G::kShort) logits();
          if (!E) dp();
          if (more) ++g;
        }
      }
      commit(on, bar(kdqDone));      // no matrix instruction is under way when the CTA ends
      wait.end(bar(kdqDone), 0);
    } else if (warp == kLoadWarp) {
      Loader<TERMS, DW> ld{lane, bar(kdqFix), wait};
      int g = 0, job = 0, issued = 0, issued_q = 0;         // tiles, and jobs with any; those whose copies the first lane has issued
      bool stop = false;          // after a failure: jobs without any tile
      for (int m = 0, index = blockIdx.x;; ++m) {
        Job j = dq_job(a, index);
        if (stop) { j.n = min(j.n, 0); j.n0 = j.n1 = 0; }
        const int kvh = j.h / a.group;
        if (!publish_job(tail, m, j, bar(kdqJob), bar(kdqJobFree), lane, wait)) break;
        if (j.n < 0) break;
        for (int i = 0; i < 2 * j.n; ++i, ++g) {
          if (i == 1) {      // behind the first tile of keys, which finds room earlier
            if (job > 0) ld.need(bar(kdqQFree), (job - 1) & 1);
            if (ld.go()) {
              tail->tiles[job & 1] = j.n;
              expect(bar(kdqQ), 2 * tile_bytes);
              ld.copies(sq, &maps.q, j.q0 + j.row0, j.h, bar(kdqQ));
              ld.copies(sg, &maps.g, j.q0 + j.row0, j.h, bar(kdqQ));
              ++issued_q;
            }
            __syncwarp();
          }
          if (g >= R) ld.need(bar(kdqEmpty + g % R), (g / R - 1) & 1);
          const int r = j.k0 + (i >> 1) * kTile;
          issued += ld.tile(ring + (g % R) * tile_bytes, (i & 1) ? &maps.v : &maps.k, j.c0 + r, kvh, bar(kdqFull + g % R), j.lk - r, !(i & 1));
        }
        job += j.n > 0;
        index = next_index(a.queue, gridDim.x, a.jobs, lane);
        stop = __any_sync(0xffffffffu, wait.failed());
      }
      // no copy is under way when the CTA ends
      if (job > 0) ld.need(bar(kdqQFree), (job - 1) & 1);
      for (int t = max(0, issued - R); t < issued; ++t) wait.end(bar(kdqFull + t % R), (t / R) & 1);
      if (issued_q > 0) wait.end(bar(kdqQ), (issued_q - 1) & 1);
      if (ld.go()) { tail->tiles[job & 1] = 0; arrive(bar(kdqQ)); }      // no more jobs
      __syncwarp();
    }
  } else {
    more_regs<kComputeRegs>();
    const int half = warp >> 2, w = warp & 3, col = 64 * half;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w) << 16), c2 = col / 2;
    const Packed to = E ? Packed{{kDs + c2, kDs + 64 + c2, kDs + 128 + c2}, {}} : Packed{{kDs + (uint32_t)col, kDs + 32 + (uint32_t)col, 256 + c2}, {}};
    const float2 scale = make_float2(a.scale_log2, a.scale_log2);
    // a row's statistics, and the power of two of its dS; rows that are not there: exp(-inf) = 0
    auto stats = [&](const Job& j, float& e, float& delta, int& shift) {
      const int row = j.row0 + w * 32 + lane;
      e = -INFINITY; delta = 0.f; shift = 0;
      if (j.n >= 0 && row < j.lq) {
        const long long at = (long long)j.h * a.nq + j.q0 + row;
        if constexpr (kShifted<T>) shift = grad_shift(a.size_g[at], j.size_v);
        e = (float)shift - a.lse[at]; delta = a.delta[at];
      }
    };
    int g = 0, job = 0;
    Job j = take_job(tail, 0, bar(kdqJob), bar(kdqJobFree), lane, wait);
    float e, delta;
    int shift;
    stats(j, e, delta, shift);
    for (int m = 1; j.n >= 0; ++m) {
      const int row = j.row0 + w * 32 + lane, first = j.row0 + w * 32;
      const int off = j.lk - j.lq;
      const int lim = min(a.causal ? row + off : j.lk - 1, j.lk - 1), lim_first = min(a.causal ? first + off : j.lk - 1, j.lk - 1);
      const bool there = row < j.lq;
      constexpr int kOwn = TERMS == 1 ? 1 : DW / 2;
      float own[kOwn];                         // dq so far (float32), half of the row
#pragma unroll
      for (int c = 0; c < kOwn; ++c) own[c] = 0.f;
      const float2 ref = make_float2(e, e);
      for (int i = 0; i < j.n; ++i, ++g) {
        uint32_t x[64], y[64];
        wait(bar(kdqS), g & 1);
        fence_after();
        ld32(lanes + col, x);
        ld32(lanes + col + 32, x + 32);
        wait_ld(x);
        fence_before();
        arrive(bar(kdqSRead));
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
          pow2_16<TERMS == 1>(x + c, scale, ref, v);
#pragma unroll
          for (int q = 0; q < 16; ++q) x[c + q] = __float_as_uint(v[q]);
        }
        const int kb = j.k0 + i * kTile + col;
        wait(bar(kdqDp), g & 1);
        fence_after();
        ld32(lanes + kTile + col, y);
        ld32(lanes + kTile + col + 32, y + 32);
        wait_ld(y);
        if (E) {
          fence_before();
          arrive(bar(kdqDpRead));
          if (g > 0) { wait(bar(kdqDsDone), (g - 1) & 1); fence_after(); }
        }
        if constexpr (TERMS == 3) { if (i > 0) add_cols<DW, DW / 2>(lanes + kOut + half * (DW / 2), own); }
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * (__uint_as_float(y[c]) - delta));
        if (kb + 63 > lim_first) {
#pragma unroll
          for (int c = 0; c < 64; ++c) if (kb + c > lim) x[c] = 0;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(x[c + q]);
          put16<M, TERMS>(to, lanes, c, v);
        }
        wait_st();
        fence_before();
        arrive(bar(kdqDs));
      }
      const Job after = take_job(tail, m, bar(kdqJob), bar(kdqJobFree), lane, wait);
      const float f0 = kShifted<T> ? a.scale * two_to(-shift) : a.scale;
      stats(after, e, delta, shift);
      if (j.n > 0) {
        wait(bar(kdqOut), job & 1);
        fence_after();
      }
      const float f = wait.failed() ? NAN : f0;
      const long long at_row = ((long long)(j.q0 + row) * a.hq + j.h) * d;
      auto put = [&](auto* dst) {
        if constexpr (TERMS == 3) {
          if (j.n > 0) add_cols<DW, DW / 2>(lanes + kOut + half * (DW / 2), own);
#pragma unroll
          for (int c = 0; c < kOwn; ++c) own[c] *= f;
#pragma unroll
          for (int c = 0; c < kOwn; c += 16) if (there && half * kOwn + c < d) store16(dst + half * kOwn + c, own + c);
        } else {
          for (int c = 16 * half; c < d; c += 32) {
            uint32_t o[16];
            float v[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) o[q] = 0;
            if (j.n > 0) { ld16(lanes + kOut + c, o); wait_ld(o); }
#pragma unroll
            for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(o[q]) * f;
            if (there) store16(dst + c, v);
          }
        }
      };
      if (a.pieces > 1) put(a.share[0] + (long long)j.piece * a.nq * a.hq * d + at_row);
      else put(static_cast<T*>(a.dq) + at_row);
      if (j.n > 0) ++job;      // read before the next job's dS are handed over, and only then written again
      j = after;
    }
    fence_before();
  }
  __syncthreads();
  if (tid == 0) wait.report(a.error);
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem); }
}

// dk and dv: 128 keys of one key head.  Rows of the products are keys, columns the queries of all heads of the group, 128 at a time.  Tensor memory:
// logits at 0 (P replaces them), dP at 128 (dS replaces it), dv at 256, dk at 384 (float32: the third terms of P and dS at 256 and 320, dv
// at 384, dk at 448; up to 64 values a head in 16 bits: P at 256, dS at 320, dv at 384, dk at 448).  The tensor cores work in the order
// dv(i), logits(i + 1), dk(i), dP(i + 1): each pair runs beside the other half of the elementwise work.
enum DkvBar { kkvFull, kkvEmpty = kkvFull + 8, kkvK = kkvEmpty + 8, kkvKFree, kkvS, kkvP, kkvDp, kkvDs, kkvOut, kkvFix, kkvDone, kkvStat, kkvStatFree = kkvStat + 2,
              kkvSRead = kkvStatFree + 2, kkvDpRead, kkvPDone, kkvDsDone, kkvJob, kkvJobFree = kkvJob + 2, kDkvBars = kkvJobFree + 2 };
__device__ __forceinline__ Job dkv_job(const PackedArgs& a, int index) {
  Job j = {};
  j.n = -1;
  if (index >= a.jobs) return j;
  const int unit = index / a.pieces;
  const int4 item = __ldg(a.items + unit / a.hk);
  j.piece = index % a.pieces; j.h = unit % a.hk;
  j.q0 = __ldg(a.start_q + item.x); j.lq = __ldg(a.start_q + item.x + 1) - j.q0; j.c0 = __ldg(a.start_kv + item.x); j.lk = __ldg(a.start_kv + item.x + 1) - j.c0;
  j.row0 = item.y * kTile; j.i0 = item.z;
  j.per = (max(j.lq - j.i0, 0) + kTile - 1) / kTile;
  if (a.largest) {
    const unsigned* most = a.largest + ((long long)item.x * a.hk + j.h) * 2;
    j.shift = grad_shift(__uint_as_float(__ldg(most)), __uint_as_float(__ldg(most + 1)));
  }
  const int all = j.per * a.group, share = all / a.pieces, more = all % a.pieces;
  j.j0 = j.piece * share + min(j.piece, more); j.n = share + (j.piece < more);
  return j;
}

template <typename T, int TERMS, int DW>
__global__ void __launch_bounds__(kThreads, 1) dkv_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  using M = typename Operand<T, TERMS>::type;
  using G = Geometry<TERMS, DW>;
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d;
  constexpr int tile_bytes = G::kSubs * (int)G::kSub, R = G::kRing;
  float* stats = reinterpret_cast<float*>(smem + (2 + R) * tile_bytes);      // [2][128] -lse in log2, [2][128] -delta
  Tail* tail = reinterpret_cast<Tail*>(stats + 4 * kTile);
  const uint32_t sk = smem_addr(smem), sv = sk + tile_bytes, ring = sv + tile_bytes, bar0 = smem_addr(tail->bars);
  const Wait wait{smem_addr(&tail->failed), a.wait_tries};
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kDkvBars; ++i)
      init_bar(bar(i), i == kkvP || i == kkvDs || i == kkvSRead || i == kkvDpRead ? 256
                       : i == kkvStat || i == kkvStat + 1 ? 64 : i == kkvStatFree || i == kkvStatFree + 1 ? 8 : i >= kkvJobFree ? 10 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;
  constexpr bool E = G::kEarly;
  constexpr uint32_t kP = E ? 256 : 0, kDs = E ? 320 : kTile, kDv = E || TERMS == 3 ? 384 : 256, kDk = E || TERMS == 3 ? 448 : 384;

  // tiles (queries 0, 2, .., cotangents 1, 3, ..) and jobs with any are counted as in dq_kernel
  if (warp >= kMmaWarp) {
    fewer_regs<kOtherRegs>();
    if (warp == kMmaWarp) {
      const uint32_t on = elect_one();
      auto need = [&](uint32_t b, uint32_t parity) { wait(b, parity); fence_after(); };
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };
      auto ready = [&](int j) { need(bar(kkvFull + j % R), (j / R) & 1); };
      auto give = [&](int j) { commit(on, bar(kkvEmpty + j % R)); };
      auto packed_at = [&](uint32_t at, uint32_t third) { return E ? Packed{{at}, {32}} : Packed{{at, at + 32, third}, {64, 64, 32}}; };
      int g = -1;
      for (int job = 0;; ++job) {
        need(bar(kkvK), job & 1);
        const int n = __shfl_sync(0xffffffffu, wait.failed() ? 0 : tail->tiles[job & 1], 0);
        if (n == 0) break;
        for (int i = -1; i < n; ++i) {
          const bool more = i + 1 < n;
          auto logits = [&] {
            if (!more) return;
            ready(2 * g + 2);
            if (E && g >= 0) need(bar(kkvSRead), g & 1);
            product_rows<M, TERMS, DW>(on, tmem, sk, slot(2 * g + 2), d);
            commit(on, bar(kkvS));
          };
          auto dp = [&] {
            if (!more) return;
            ready(2 * g + 3);
            if (E && g >= 0) need(bar(kkvDpRead), g & 1);
            product_rows<M, TERMS, DW>(on, tmem + kTile, sv, slot(2 * g + 3), d);
            commit(on, bar(kkvDp));
            if (i + 2 == n) commit(on, bar(kkvKFree));
          };
          if (E) logits();
          if (i >= 0) {
            need(bar(kkvP), g & 1);
            product_cols<M, TERMS, DW>(on, tmem + kDv, packed_at(tmem + kP, tmem + 256), slot(2 * g + 1), d, i > 0);
            if (E) commit(on, bar(kkvPDone));
            give(2 * g + 1);
          }
          if (!E && !G::kShort) logits();
          if (E) dp();
          if (i >= 0) {
            need(bar(kkvDs), g & 1);
            product_cols<M, TERMS, DW>(on, tmem + kDk, packed_at(tmem + kDs, tmem + 320), slot(2 * g), d, i > 0);
            if (E) commit(on, bar(kkvDsDone));
            if (!more) commit(on, bar(kkvOut));
            give(2 * g);
          }
          if (G::kShort) logits();
          if (!E) dp();
          if (more) ++g;
        }
      }
      commit(on, bar(kkvDone));      // no matrix instruction is under way when the CTA ends
      wait.end(bar(kkvDone), 0);
    } else if (warp == kLoadWarp) {
      Loader<TERMS, DW> ld{lane, bar(kkvFix), wait};
      int g = 0, job = 0, issued = 0, issued_k = 0;         // as in dq_kernel
      bool stop = false;
      for (int m = 0, index = blockIdx.x;; ++m) {
        Job j = dkv_job(a, index);
        if (stop) { j.n = min(j.n, 0); j.n0 = j.n1 = 0; }
        if (!publish_job(tail, m, j, bar(kkvJob), bar(kkvJobFree), lane, wait)) break;
        if (j.n < 0) break;
        for (int i = 0; i < 2 * j.n; ++i, ++g) {
          if (i == 1) {
            if (job > 0) ld.need(bar(kkvKFree), (job - 1) & 1);
            if (ld.go()) {
              tail->tiles[job & 1] = j.n;
              expect(bar(kkvK), 2 * tile_bytes);
              ld.copies(sk, &maps.k, j.c0 + j.row0, j.h, bar(kkvK));
              ld.copies(sv, &maps.v, j.c0 + j.row0, j.h, bar(kkvK));
              ++issued_k;
            }
            __syncwarp();
          }
          if (g >= R) ld.need(bar(kkvEmpty + g % R), (g / R - 1) & 1);
          const int t = j.j0 + (i >> 1), hq = j.h * a.group + t / j.per, b = j.i0 + (t % j.per) * kTile;
          issued += ld.tile(ring + (g % R) * tile_bytes, (i & 1) ? &maps.g : &maps.q, j.q0 + b, hq, bar(kkvFull + g % R), j.lq - b, true);
        }
        job += j.n > 0;
        index = next_index(a.queue + 1, gridDim.x, a.jobs, lane);
        stop = __any_sync(0xffffffffu, wait.failed());
      }
      if (job > 0) ld.need(bar(kkvKFree), (job - 1) & 1);
      for (int t = max(0, issued - R); t < issued; ++t) wait.end(bar(kkvFull + t % R), (t / R) & 1);
      if (issued_k > 0) wait.end(bar(kkvK), (issued_k - 1) & 1);
      if (ld.go()) { tail->tiles[job & 1] = 0; arrive(bar(kkvK)); }      // no more jobs
      __syncwarp();
    } else {
      const int r0 = (warp - kLoadWarp - 1) * 32 + lane;
      int g = 0;
      for (int m = 0;; ++m) {
        const Job j = take_job(tail, m, bar(kkvJob), bar(kkvJobFree), lane, wait);
        if (j.n < 0) break;
        const float un = kShifted<T> ? packed::prob_unscale<T>() * two_to(j.shift) : 1.f;
        for (int i = 0; i < j.n; ++i, ++g) {
          const int st = g & 1, hq = j.h * a.group + (j.j0 + i) / j.per, b = j.i0 + ((j.j0 + i) % j.per) * kTile;
          if (g >= 2) wait(bar(kkvStatFree + st), ((g >> 1) - 1) & 1);
          for (int r = r0; r < kTile; r += 64) {
            const bool ok = b + r < j.lq;
            const long long at = (long long)hq * a.nq + j.q0 + b + r;
            stats[st * kTile + r] = ok ? packed::prob_shift<T>() - a.lse[at] : -INFINITY;
            stats[(2 + st) * kTile + r] = ok ? -a.delta[at] * un : 0.f;
          }
          arrive(bar(kkvStat + st));
        }
      }
    }
  } else {
    more_regs<kComputeRegs>();
    const int half = warp >> 2, w = warp & 3, col = 64 * half;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w) << 16), c2 = col / 2;
    const Packed to_p = E ? Packed{{kP + c2}, {}} : Packed{{kP + (uint32_t)col, kP + 32 + (uint32_t)col, 256 + c2}, {}};
    const Packed to_s = E ? Packed{{kDs + c2}, {}} : Packed{{kDs + (uint32_t)col, kDs + 32 + (uint32_t)col, 320 + c2}, {}};
    const float2 scale = make_float2(a.scale_log2, a.scale_log2);
    int g = 0, job = 0;
    Job j = take_job(tail, 0, bar(kkvJob), bar(kkvJobFree), lane, wait);
    for (int m = 1; j.n >= 0; ++m) {
      const int row = j.row0 + w * 32 + lane, last = j.row0 + w * 32 + 31;
      // first query that sees this key, and that sees the warp's last key
      const int off = j.lk - j.lq, lim = a.causal ? row - off : 0, lim_last = a.causal ? last - off : 0;
      constexpr int kOwn = TERMS == 1 ? 1 : DW / 2;
      float own[2][kOwn];                      // dv, dk so far (float32), half of the row
#pragma unroll
      for (int c = 0; c < kOwn; ++c) own[0][c] = own[1][c] = 0.f;
      const float un = kShifted<T> ? packed::prob_unscale<T>() * two_to(j.shift) : 1.f;      // from 2^15 P to P times the power of dS
      for (int i = 0; i < j.n; ++i, ++g) {
        const int st = g & 1, ib = j.i0 + ((j.j0 + i) % j.per) * kTile + col;
        uint32_t x[64], y[64];
        wait(bar(kkvStat + st), (g >> 1) & 1);
        wait(bar(kkvS), g & 1);
        fence_after();
        ld32(lanes + col, x);
        ld32(lanes + col + 32, x + 32);
        wait_ld(x);
        if (E) { fence_before(); arrive(bar(kkvSRead)); }
        if constexpr (TERMS == 3) { if (i > 0) add_cols<DW, DW / 2>(lanes + kDv + half * (DW / 2), own[0]); }
        const float4* e = reinterpret_cast<const float4*>(stats + st * kTile + col);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float4 v = e[c];
          const float2 z0 = __ffma2_rn(make_float2(__uint_as_float(x[4 * c]), __uint_as_float(x[4 * c + 1])), scale, make_float2(v.x, v.y));
          const float2 z1 = __ffma2_rn(make_float2(__uint_as_float(x[4 * c + 2]), __uint_as_float(x[4 * c + 3])), scale, make_float2(v.z, v.w));
          const float2 r1 = TERMS == 1 ? pow2_poly(z1) : make_float2(pow2(z1.x), pow2(z1.y));
          x[4 * c] = __float_as_uint(pow2(z0.x)); x[4 * c + 1] = __float_as_uint(pow2(z0.y));
          x[4 * c + 2] = __float_as_uint(r1.x); x[4 * c + 3] = __float_as_uint(r1.y);
        }
        if (E && g > 0) { wait(bar(kkvPDone), (g - 1) & 1); fence_after(); }
        if (a.causal && ib < lim_last) {
#pragma unroll
          for (int c = 0; c < 64; ++c) if (ib + c < lim) x[c] = 0;
        }
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(x[c + q]);
          put16<M, TERMS>(to_p, lanes, c, v);
        }
        wait_st();
        fence_before();
        arrive(bar(kkvP));
        wait(bar(kkvDp), g & 1);
        fence_after();
        ld32(lanes + kTile + col, y);
        ld32(lanes + kTile + col + 32, y + 32);
        wait_ld(y);
        if (E) {
          fence_before();
          arrive(bar(kkvDpRead));
          if (g > 0) { wait(bar(kkvDsDone), (g - 1) & 1); fence_after(); }
        }
        if constexpr (TERMS == 3) { if (i > 0) add_cols<DW, DW / 2>(lanes + kDk + half * (DW / 2), own[1]); }
        const float4* dl = reinterpret_cast<const float4*>(stats + (2 + st) * kTile + col);
#pragma unroll
        for (int c = 0; c < 64; c += 16) {
          float v[16];
#pragma unroll
          for (int q = 0; q < 16; q += 4) {
            const float4 z = dl[(c + q) / 4];
            v[q] = __uint_as_float(x[c + q]) * fmaf(__uint_as_float(y[c + q]), un, z.x);
            v[q + 1] = __uint_as_float(x[c + q + 1]) * fmaf(__uint_as_float(y[c + q + 1]), un, z.y);
            v[q + 2] = __uint_as_float(x[c + q + 2]) * fmaf(__uint_as_float(y[c + q + 2]), un, z.z);
            v[q + 3] = __uint_as_float(x[c + q + 3]) * fmaf(__uint_as_float(y[c + q + 3]), un, z.w);
          }
          put16<M, TERMS>(to_s, lanes, c, v);
        }
        __syncwarp();
        if (lane == 0) arrive(bar(kkvStatFree + st));
        wait_st();
        fence_before();
        arrive(bar(kkvDs));
      }
      const Job after = take_job(tail, m, bar(kkvJob), bar(kkvJobFree), lane, wait);
      if (j.n > 0) {
        wait(bar(kkvOut), job & 1);
        fence_after();
      }
      const bool there = row < j.lk, bad = wait.failed();
      const long long at = ((long long)(j.c0 + row) * a.hk + j.h) * d;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float f = bad ? NAN : !which ? packed::prob_unscale<T>() : kShifted<T> ? a.scale * two_to(-j.shift) : a.scale;
        const uint32_t from = lanes + (which ? kDk : kDv);
        auto put = [&](auto* dst) {
          if constexpr (TERMS == 3) {
            if (j.n > 0) add_cols<DW, DW / 2>(from + half * (DW / 2), own[which]);
#pragma unroll
            for (int c = 0; c < kOwn; ++c) own[which][c] *= f;
#pragma unroll
            for (int c = 0; c < kOwn; c += 16) if (there && half * kOwn + c < d) store16(dst + half * kOwn + c, own[which] + c);
          } else {
            for (int c = 16 * half; c < d; c += 32) {
              uint32_t o[16];
              float v[16];
#pragma unroll
              for (int q = 0; q < 16; ++q) o[q] = 0;
              if (j.n > 0) { ld16(from + c, o); wait_ld(o); }
#pragma unroll
              for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(o[q]) * f;
              if (there) store16(dst + c, v);
            }
          }
        };
        if (a.pieces > 1) put(a.share[which ? 1 : 2] + (long long)j.piece * a.nkv * a.hk * d + at);
        else put(static_cast<T*>(which ? a.dk : a.dv) + at);
      }
      if (j.n > 0) ++job;      // read before the next job's P are handed over, and only then written again
      j = after;
    }
    fence_before();
  }
  __syncthreads();
  if (tid == 0) wait.report(a.error);
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem); }
}

static_assert(kFwdBars <= kBars && kDqBars <= kBars && kDkvBars <= kBars, "barriers");

// float32 rows -> three bfloat16 terms, (rows, heads, 3, DW), zeros behind d; a thread per eight values, up to four operands
struct SplitArgs { Rows src[4]; __nv_bfloat16* dst[4]; int rows[4], heads[4]; };
template <int DW>
__global__ void __launch_bounds__(256) split_kernel(const SplitArgs A, int d) {
  const int o = blockIdx.y;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x, hr = e / (DW / 8);
  const int part = (int)(e % (DW / 8)) * 8;
  if (hr >= (long long)A.rows[o] * A.heads[o]) return;
  const long long r = hr / A.heads[o];
  const int h = (int)(hr % A.heads[o]);
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.f;
  if (part < d) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(A.src[o].p) + r * A.src[o].row + h * A.src[o].head + part);
    const float4 x = p[0], y = p[1];
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
  }
#pragma unroll
  for (int term = 0; term < 3; ++term) {
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u[k] = packed::Half<__nv_bfloat16>::pack(v[2 * k], v[2 * k + 1]);
      const float2 f = packed::Half<__nv_bfloat16>::unpack(u[k]);
      v[2 * k] -= f.x; v[2 * k + 1] -= f.y;
    }
    *reinterpret_cast<uint4*>(A.dst[o] + (hr * 3 + term) * DW + part) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
Encode encoder() {
  static const Encode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return fn;
}
// (values, rows, heads) of 16-bit values; boxes of `width` values x 128 rows, a row as long as the swizzle
bool map_of(CUtensorMap* m, bool bf16, const Rows& r, long long rows, int heads, int d, int width) {
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)heads};
  const cuuint64_t strides[2] = {(cuuint64_t)r.row * 2, (cuuint64_t)r.head * 2};
  const cuuint32_t box[3] = {(cuuint32_t)width, kTile, 1}, ones[3] = {1, 1, 1};
  return encoder()(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(r.p), dims, strides, box, ones,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <typename T, int TERMS, int DW> int maps_of(Maps* m, cudaStream_t st, const PackedArgs& a, bool reverse, void* workspace) {
  if (!encoder()) return kCudaError;
  // Encoding a map goes to the driver, which wants the device's context current on this thread; the runtime makes it so at a thread's first
  // call that needs it, and autograd's threads may come here first.
  int device = 0;
  SO3LR_CUDA_CHECK(cudaGetDevice(&device));
  SO3LR_CUDA_CHECK(cudaSetDevice(device));
  CUtensorMap* maps[4] = {&m->q, &m->k, &m->v, &m->g};
  const Rows rows[4] = {a.q, a.k, a.v, a.g};
  const int n[4] = {a.nq, a.nkv, a.nkv, a.nq}, heads[4] = {a.hq, a.hk, a.hk, a.hq}, operands = reverse ? 4 : 3;
  if constexpr (TERMS == 1) {
    for (int i = 0; i < operands; ++i)
      if (!map_of(maps[i], std::is_same<T, __nv_bfloat16>::value, rows[i], n[i], heads[i], a.d, 64)) return kInvalidArgument;
  } else {
    SplitArgs A;
    __nv_bfloat16* at = static_cast<__nv_bfloat16*>(workspace);
    long long most = 0;
    for (int i = 0; i < operands; ++i) {
      A.src[i] = rows[i]; A.dst[i] = at; A.rows[i] = n[i]; A.heads[i] = heads[i];
      const long long values = (long long)n[i] * heads[i] * 3 * DW;
      if (!map_of(maps[i], true, Rows{at, (long long)heads[i] * 3 * DW, DW}, n[i], 3 * heads[i], DW, DW)) return kInvalidArgument;
      at += values;
      most = std::max(most, values);
    }
    split_kernel<DW><<<dim3((unsigned)((most / 24 + 255) / 256), operands), 256, 0, st>>>(A, a.d);
    count_launch();
  }
  if (!reverse) m->g = m->q;
  return kOk;
}
template <int TERMS, int DW> constexpr int reverse_smem(bool stats) {
  using G = Geometry<TERMS, DW>;
  return 1024 + (2 + G::kRing) * G::kSubs * (int)G::kSub + (stats ? 4 * kTile * 4 : 0) + (int)sizeof(Tail);
}
template <auto kernel> int launch(int64_t grid, int threads, int smem, cudaStream_t st, const PackedArgs& a, const Maps& m) {
  packed::allow_smem<kernel>(smem);
  if (grid > 0x7fffffff) return kTooLarge;
  kernel<<<(unsigned)grid, threads, smem, st>>>(a, m);
  count_launch();
  return kOk;
}
// up to `ctas` CTAs, which work through `jobs`
template <auto kernel> int launch_jobs(int64_t jobs, int64_t ctas, int threads, int smem, cudaStream_t st, PackedArgs a, const Maps& m) {
  if (jobs > 0x7fff0000) return kTooLarge;
  a.jobs = (int)jobs;
  return launch<kernel>(std::min(jobs, ctas), threads, smem, st, a, m);
}
template <typename T, int TERMS, int DW, int TILES> int forward_of(cudaStream_t st, PackedArgs a, int n_items, const PackedPieces& pieces, void* workspace) {
  Maps m;
  int rc = maps_of<T, TERMS, DW>(&m, st, a, false, workspace);
  if (rc) return rc;
  a.pieces = pieces.forward;
  if (a.pieces > 1) {
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + (TERMS == 3 ? packed_split_bytes(a.nq, a.nkv, a.hq, a.hk, a.d, false) : 0));
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (long long)a.pieces * a.nq * a.hq * a.d);
  }
  using F = Forward<TERMS, DW, TILES>;
  const int64_t jobs = (int64_t)n_items * a.hq * a.pieces, ctas = F::kQueued ? sm_count() * (TILES == 1 ? 2 : 1) : jobs;
  if (jobs <= ctas) a.queue = nullptr;      // each CTA's first job is all
  else SO3LR_CUDA_CHECK(cudaMemsetAsync(a.queue, 0, sizeof(int), st));
  rc = launch_jobs<forward_kernel<T, TERMS, DW, TILES>>(jobs, ctas, F::kThreads, F::kSmem, st, a, m);
  if (rc || a.pieces == 1) return rc;
  return packed_join<T>(st, a);
}
template <typename T, int TERMS, int DW>
int reverse_of(cudaStream_t st, PackedArgs a, const int4* items_q, int n_q, const int4* items_kv, int n_kv, const PackedPieces& pieces, void* workspace) {
  Maps m;
  int rc = maps_of<T, TERMS, DW>(&m, st, a, true, workspace);
  if (rc) return rc;
  const long long stride_q = (long long)a.nq * a.hq * a.d, stride_kv = (long long)a.nkv * a.hk * a.d;
  float* share = reinterpret_cast<float*>(static_cast<char*>(workspace) + (TERMS == 3 ? packed_split_bytes(a.nq, a.nkv, a.hq, a.hk, a.d, true) : 0));
  if (pieces.dq > 1) { a.share[0] = share; share += pieces.dq * stride_q; }
  if (pieces.dkv > 1) { a.share[1] = share; a.share[2] = share + pieces.dkv * stride_kv; }
  a.items = items_q;
  a.pieces = pieces.dq;
  rc = launch_jobs<dq_kernel<T, TERMS, DW>>((int64_t)n_q * a.hq * a.pieces, sm_count(), kThreads, reverse_smem<TERMS, DW>(false), st, a, m);
  if (rc) return rc;
  a.items = items_kv;
  a.pieces = pieces.dkv;
  rc = launch_jobs<dkv_kernel<T, TERMS, DW>>((int64_t)n_kv * a.hk * a.pieces, sm_count(), kThreads, reverse_smem<TERMS, DW>(true), st, a, m);
  if (rc || (pieces.dq == 1 && pieces.dkv == 1)) return rc;
  return packed_sum<T>(st, a, pieces.dq, pieces.dkv);
}

}  // namespace

template <typename T> int packed_forward_tc(cudaStream_t st, PackedArgs a, int n_items, const PackedPieces& pieces, void* workspace) {
  const bool one = packed_one_tile(sizeof(T) == 4, a.d, a.longest_kv);
  if constexpr (sizeof(T) == 2) {
    if (a.d > 64) return one ? forward_of<T, 1, 128, 1>(st, a, n_items, pieces, workspace) : forward_of<T, 1, 128, 2>(st, a, n_items, pieces, workspace);
    return forward_of<T, 1, 64, 1>(st, a, n_items, pieces, workspace);
  } else {
    if (a.d > 32) return forward_of<T, 3, 64, 2>(st, a, n_items, pieces, workspace);
    return one ? forward_of<T, 3, 32, 1>(st, a, n_items, pieces, workspace) : forward_of<T, 3, 32, 2>(st, a, n_items, pieces, workspace);
  }
}
template <typename T>
int packed_reverse_tc(cudaStream_t st, PackedArgs a, const int4* items_q, int n_q, const int4* items_kv, int n_kv, const PackedPieces& pieces, void* workspace) {
  if constexpr (sizeof(T) == 2) return a.d <= 64 ? reverse_of<T, 1, 64>(st, a, items_q, n_q, items_kv, n_kv, pieces, workspace)
                                                 : reverse_of<T, 1, 128>(st, a, items_q, n_q, items_kv, n_kv, pieces, workspace);
  else return a.d <= 32 ? reverse_of<T, 3, 32>(st, a, items_q, n_q, items_kv, n_kv, pieces, workspace)
                        : reverse_of<T, 3, 64>(st, a, items_q, n_q, items_kv, n_kv, pieces, workspace);
}
// A word of host memory for every device, which a kernel sets when a wait has run out: the next call finds it without waiting for the device.
int packed_error_word(int** word) {
  static std::mutex lock;
  static int* words[64] = {};
  int dev = 0;
  SO3LR_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return kInvalidArgument;
  const std::lock_guard<std::mutex> held(lock);
  if (!words[dev]) {
    // the first call of all may come while its stream is being captured
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    SO3LR_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
    cudaThreadExchangeStreamCaptureMode(&mode);
    SO3LR_CUDA_CHECK(e);
    words[dev] = static_cast<int*>(p);
    __atomic_store_n(words[dev], 0, __ATOMIC_RELAXED);
  }
  *word = words[dev];
  return kOk;
}

template int packed_forward_tc<__nv_bfloat16>(cudaStream_t, PackedArgs, int, const PackedPieces&, void*);
template int packed_reverse_tc<__nv_bfloat16>(cudaStream_t, PackedArgs, const int4*, int, const int4*, int, const PackedPieces&, void*);
template int packed_forward_tc<__half>(cudaStream_t, PackedArgs, int, const PackedPieces&, void*);
template int packed_reverse_tc<__half>(cudaStream_t, PackedArgs, const int4*, int, const int4*, int, const PackedPieces&, void*);
template int packed_forward_tc<float>(cudaStream_t, PackedArgs, int, const PackedPieces&, void*);
template int packed_reverse_tc<float>(cudaStream_t, PackedArgs, const int4*, int, const int4*, int, const PackedPieces&, void*);

}  // namespace so3lr
