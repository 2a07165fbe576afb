// Attention inside the structures of a packed batch on the warp-level matrix instructions: forward, its form split over the keys, and the
// two halves of the reverse pass, for float32, bfloat16 and float16 and up to 128 values a head.
//
//   s_ij = scale q_i . k_j,  o_i = sum_j exp(s_ij - lse_i) v_j            one pass over the keys with a running maximum m and sum l:
//   a tile of keys raises m to m', o and l are scaled by exp(m - m') and the tile's share is added; o / l at the end.
//   reverse: P_ij = exp(s_ij - lse_i), dP_ij = g_i . v_j, dS_ij = P_ij (dP_ij - delta_i), delta_i = g_i . o_i,
//   dq_i = scale sum_j dS_ij k_j     (a CTA per tile of queries, walking over the keys)
//   dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij g_i   (a CTA per tile of keys, walking over the queries of all heads of its group)
// Two kernels form the exponentials twice, but every sum has one owner: no atomics, results do not change from run to run, and the
// gradients of shared keys need no second pass.
//
// A CTA has four warps with 16 rows each, or one where all structures are short (a CTA per 16 rows and head: no warp is without rows, and many
// CTAs hide each other's start); the tile of the other side is double-buffered by 16-byte asynchronous copies that fill rows and
// columns that are not there with zeros.  The accumulator fragment of one product is the A fragment of the next, so P and dS never leave
// the registers (and are rounded to the inputs' type on the way into the second product: their error then is that of one rounding of an
// input; float16 takes a power of two out of both, see kHead, prob_shift and grad_shift).  float32 runs as three products of operands split into
// two tf32 numbers each (hi hi + hi lo + lo hi): 2^-21 of the product, where a single tf32 product has 2^-11.
#pragma once
#include <atomic>

#include "packed_attention.h"

namespace so3lr {
namespace packed {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros where `ok` is false
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// x = hi + lo, hi rounded to the 11 bits of tf32 in integer arithmetic (the conversion instruction runs at an eighth of its rate); lo is exact,
// and the matrix instruction reads its upper 11 bits
__device__ __forceinline__ void tf32_split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}

template <typename T> struct Half;
// float16 keeps its 11 bits down to 2^-14 only, and a normalised probability over thousands of keys lies there: the kernels of dk and dv form
// 2^15 P (at most 2^15 < 65504, exact, no instruction more) and take the factor out of dv at the end and out of dP - delta.  dS has a
// power of two of its own (grad_shift).
template <typename T> constexpr float prob_shift() { return std::is_same<T, __half>::value ? 15.f : 0.f; }
template <typename T> constexpr float prob_unscale() { return std::is_same<T, __half>::value ? 1.f / 32768.f : 1.f; }
template <> struct Half<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
};
template <> struct Half<__half> {
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
};

// Tiles in shared memory: rows of DP values plus 16 bytes, which puts the 16-byte pieces of eight consecutive rows into different banks.
template <typename T, int DP> struct Tile {
  static constexpr int kStride = DP * (int)sizeof(T) + 16;   // bytes
  static constexpr int kChunks = DP * (int)sizeof(T) / 16;
  static constexpr int kPer = 16 / (int)sizeof(T);           // values of a chunk
};

// rows [r0, r0 + N) of one head into a tile; row r is there where r < r1
template <typename T, int DP, int N, int THREADS>
__device__ __forceinline__ void load_rows(uint32_t tile, const Rows& src, int head, long long base, int r0, int r1, int d, int tid) {
  using L = Tile<T, DP>;
  const T* p = static_cast<const T*>(src.p) + head * src.head;
#pragma unroll
  for (int i = tid; i < N * L::kChunks; i += THREADS) {
    const int r = i / L::kChunks, c = i % L::kChunks;
    const bool ok = r0 + r < r1 && c * L::kPer < d;
    copy16(tile + r * L::kStride + c * 16, ok ? p + (base + r0 + r) * src.row + c * L::kPer : p, ok);
  }
}

// ---- products of a warp's 16 rows -----------------------------------------------------------------------------------
// The tensor cores cut what they add to an accumulator to its 24 bits instead of rounding it, which shrinks a long sum by up to 2^-24 a step.
// With 16-bit operands that does not show; float32 products keep the cross terms apart from the large ones, and start every tile of the
// walked side in fresh accumulators that are added in ordinary arithmetic: at 5,000 keys 3.5e-5 of the result without, below 1e-6 with it.

// acc[16 x 8 NT] = A[16 x DP] B[8 NT x DP]^T, A at `a` (the warp's first row), B at `b`; columns from `cols` on are not needed
template <typename T, int DP, int NT, bool PART>
__device__ __forceinline__ void product_nt_of(float (&acc)[NT][4], uint32_t a, uint32_t b, int lane, int cols) {
  using L = Tile<T, DP>;
  const uint32_t al = a + (lane & 15) * L::kStride + (lane >> 4) * 16;
  const uint32_t bl = b + ((lane & 7) + ((lane >> 4) << 3)) * L::kStride + ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      uint32_t fa[4];
      ldsm4(al + ks * 32, fa);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        if (!PART || n * 8 < cols) {
          uint32_t fb[4];
          ldsm4(bl + n * 8 * L::kStride + ks * 32, fb);
          Half<T>::mma(acc[n], fa, fb);
          Half<T>::mma(acc[n + 1], fa, fb + 2);
        }
      }
    }
  } else {
    float cross[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) cross[n][0] = cross[n][1] = cross[n][2] = cross[n][3] = 0.f;
#pragma unroll 4
    for (int ks = 0; ks < DP / 8; ++ks) {
      uint32_t fa[4], ah[4], alo[4];
      ldsm4(al + ks * 32, fa);
#pragma unroll
      for (int i = 0; i < 4; ++i) tf32_split(__uint_as_float(fa[i]), ah[i], alo[i]);
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        if (!PART || n * 8 < cols) {
          uint32_t fb[4], bh[4], blo[4];
          ldsm4(bl + n * 8 * L::kStride + ks * 32, fb);
#pragma unroll
          for (int i = 0; i < 4; ++i) tf32_split(__uint_as_float(fb[i]), bh[i], blo[i]);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma_tf32(acc[n + h], ah, bh + 2 * h);
            mma_tf32(cross[n + h], alo, bh + 2 * h);
            mma_tf32(cross[n + h], ah, blo + 2 * h);
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) { acc[n][0] += cross[n][0]; acc[n][1] += cross[n][1]; acc[n][2] += cross[n][2]; acc[n][3] += cross[n][3]; }
  }
}

// acc[16 x DP] += A[16 x 8 NT] B[8 NT x DP], A the accumulator fragments of an earlier product, zero from column `rows` on
template <typename T, int DP, int NT, bool PART>
__device__ __forceinline__ void product_nn_of(float (&acc)[DP / 8][4], const float (&p)[NT][4], uint32_t b, int lane, int rows) {
  using L = Tile<T, DP>;
  if constexpr (sizeof(T) == 2) {
    const uint32_t bl = b + (lane & 15) * L::kStride + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      if (!PART || j * 16 < rows) {
        const uint32_t fa[4] = {Half<T>::pack(p[2 * j][0], p[2 * j][1]), Half<T>::pack(p[2 * j][2], p[2 * j][3]),
                                Half<T>::pack(p[2 * j + 1][0], p[2 * j + 1][1]), Half<T>::pack(p[2 * j + 1][2], p[2 * j + 1][3])};
#pragma unroll
        for (int n = 0; n < DP / 8; n += 2) {
          uint32_t fb[4];
          ldsm4t(bl + j * 16 * L::kStride + n * 16, fb);
          Half<T>::mma(acc[n], fa, fb);
          Half<T>::mma(acc[n + 1], fa, fb + 2);
        }
      }
    }
  } else {
    // the order of the contracted index is free: position t stands for column 2 t, position t + 4 for column 2 t + 1, which is how the
    // accumulator fragment holds them; B follows (rows 2 t and 2 t + 1: banks 8 t + g, all different)
    const uint32_t bl = b + 2 * (lane & 3) * L::kStride + (lane >> 2) * 4;
    uint32_t ah[NT][4], alo[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      tf32_split(p[j][0], ah[j][0], alo[j][0]); tf32_split(p[j][2], ah[j][1], alo[j][1]);
      tf32_split(p[j][1], ah[j][2], alo[j][2]); tf32_split(p[j][3], ah[j][3], alo[j][3]);
    }
#pragma unroll
    for (int n = 0; n < DP / 8; n += 4) {
      float t[4][4], cross[4][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) { t[m][0] = t[m][1] = t[m][2] = t[m][3] = 0.f; cross[m][0] = cross[m][1] = cross[m][2] = cross[m][3] = 0.f; }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (!PART || j * 8 < rows) {
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            float x, y;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(bl + j * 8 * L::kStride + (n + m) * 32) : "memory");
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(bl + (j * 8 + 1) * L::kStride + (n + m) * 32) : "memory");
            uint32_t bh[2], blo[2];
            tf32_split(x, bh[0], blo[0]); tf32_split(y, bh[1], blo[1]);
            mma_tf32(t[m], ah[j], bh);
            mma_tf32(cross[m], alo[j], bh);
            mma_tf32(cross[m], ah[j], blo);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        acc[n + m][0] += t[m][0] + cross[m][0]; acc[n + m][1] += t[m][1] + cross[m][1];
        acc[n + m][2] += t[m][2] + cross[m][2]; acc[n + m][3] += t[m][3] + cross[m][3];
      }
    }
  }
}

// A tile that is not full leaves out what is empty; the tests between the instructions cost a full one a fifth of its time, so it has none.
template <typename T, int DP, int NT>
__device__ __forceinline__ void product_nt(float (&acc)[NT][4], uint32_t a, uint32_t b, int lane, int cols) {
  if (cols >= 8 * NT) product_nt_of<T, DP, NT, false>(acc, a, b, lane, cols);
  else product_nt_of<T, DP, NT, true>(acc, a, b, lane, cols);
}
template <typename T, int DP, int NT>
__device__ __forceinline__ void product_nn(float (&acc)[DP / 8][4], const float (&p)[NT][4], uint32_t b, int lane, int rows) {
  if (rows >= 8 * NT) product_nn_of<T, DP, NT, false>(acc, p, b, lane, rows);
  else product_nn_of<T, DP, NT, true>(acc, p, b, lane, rows);
}

// the warp's accumulators (rows g and g + 8 of its 16, columns 8 n + 2 t, + 1) times `f` to a contiguous destination
template <typename T>
__device__ __forceinline__ void store2(T* p, float x, float y) {
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(p) = Half<T>::pack(x, y);
  else *reinterpret_cast<float2*>(p) = make_float2(x, y);
}

// x, y rounded, and what the rounding left of 16-bit types (the reverse pass forms g . o with both: with the rounded o alone its error is as
// large as that of dS itself in short structures)
template <typename T>
__device__ __forceinline__ void store_rest(T* p, T* rest, float x, float y) {
  store2(p, x, y);
  if constexpr (sizeof(T) == 2) {
    if (rest) {
      const float2 r = Half<T>::unpack(Half<T>::pack(x, y));
      store2(rest, x - r.x, y - r.y);
    }
  }
}

template <typename T, int DP, int NW> constexpr int key_tile() { return NW == 1 || (sizeof(T) == 4 && DP > 64) ? 32 : 64; }
template <typename T, int DP, int NW> int forward_smem(int stages) { return (16 * NW + 2 * stages * key_tile<T, DP, NW>()) * Tile<T, DP>::kStride; }
constexpr int kRevTile = 32;   // rows of the walked side in the reverse kernels: two accumulators of 16 x DP are held at the same time
template <typename T, int DP, int NW> int reverse_smem(int stages) { return (32 * NW + 2 * stages * kRevTile) * Tile<T, DP>::kStride + 4 * kRevTile * 4; }

// ---- forward --------------------------------------------------------------------------------------------------------
// SPLIT: rows are (token, head of the group) of ONE key head, a structure has at most 64 of them, and the item is a stretch of the keys;
// what it finds is joined by combine_kernel, or written where the structure has one stretch only.
template <typename T, int DP, bool SPLIT, int NW>
__global__ void __launch_bounds__(32 * NW) forward_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int BN = key_tile<T, DP, NW>(), NT = BN / 8, kRows = 16 * NW, kThreads = 32 * NW;
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sq = smem_addr(smem), sk = sq + kRows * L::kStride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = SPLIT ? a.hk : a.hq, piece = SPLIT ? 0 : blockIdx.x % a.pieces, index = SPLIT ? blockIdx.x : blockIdx.x / a.pieces, unit = index / heads;
  const int4 item = a.items[unit];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int G = SPLIT ? a.group : 1, hy = index % heads, kvh = SPLIT ? hy : hy / a.group;
  const int rows = lq * G, row0 = SPLIT ? 0 : item.y * kRows;
  const int share = SPLIT ? 0 : ((item.w + BN - 1) / BN + a.pieces - 1) / a.pieces * BN;      // keys of a piece
  const int k0 = SPLIT ? item.z : min(item.w, piece * share), k1 = SPLIT ? item.w : min(item.w, k0 + share);
  const int nt = (max(k1 - k0, 0) + BN - 1) / BN, stages = a.stages;
  const uint32_t sv = sk + stages * BN * L::kStride;

  {  // queries
    const T* p = static_cast<const T*>(a.q.p);
#pragma unroll 4
    for (int i = tid; i < kRows * L::kChunks; i += kThreads) {
      const int r = i / L::kChunks, c = i % L::kChunks, pr = row0 + r;
      const bool ok = pr < rows && c * L::kPer < a.d;
      const int tok = SPLIT ? pr / G : pr, head = SPLIT ? hy * G + pr % G : hy;
      copy16(sq + r * L::kStride + c * 16, ok ? p + (long long)(q0 + tok) * a.q.row + head * a.q.head + c * L::kPer : p, ok);
    }
  }
  auto load = [&](int it) {
    if (it < nt) {
      const int buf = it & (stages - 1), b = k0 + it * BN;
      load_rows<T, DP, BN, kThreads>(sk + buf * BN * L::kStride, a.k, kvh, c0, b, k1, a.d, tid);
      load_rows<T, DP, BN, kThreads>(sv + buf * BN * L::kStride, a.v, kvh, c0, b, k1, a.d, tid);
    }
    copy_commit();
  };
  load(0);

  const int wr = row0 + warp * 16, ra = wr + (lane >> 2), rb = ra + 8;      // this thread's two rows
  // last key that a row sees
  const int off = lk - lq, big = 0x7fffffff;
  const int lim_a = a.causal ? (SPLIT ? ra / G : ra) + off : big, lim_b = a.causal ? (SPLIT ? rb / G : rb) + off : big;
  const int lim_lo = a.causal ? (SPLIT ? wr / G : wr) + off : big, lim_hi = a.causal ? (SPLIT ? (wr + 15) / G : wr + 15) + off : big;
  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
  constexpr float head = kHead<T, false>;
  for (int it = 0; it < nt; ++it) {
    if (stages == 2) { load(it + 1); copy_wait<1>(); } else { if (it > 0) load(it); copy_wait<0>(); }
    __syncthreads();
    const int kb = k0 + it * BN, buf = it & (stages - 1);
    if (wr < rows && kb <= lim_hi) {
      float p[NT][4];
      const int cols = k1 - kb;
      product_nt<T, DP, NT>(p, sq + warp * 16 * L::kStride, sk + buf * BN * L::kStride, lane, cols);
      if (kb + BN > k1 || kb + BN - 1 > lim_lo) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = kb + n * 8 + 2 * (lane & 3) + e;
            if (j >= k1 || j > lim_a) p[n][e] = -INFINITY;
            if (j >= k1 || j > lim_b) p[n][2 + e] = -INFINITY;
          }
        }
      }
      float xa = p[0][0], xb = p[0][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) { xa = fmaxf(xa, fmaxf(p[n][0], p[n][1])); xb = fmaxf(xb, fmaxf(p[n][2], p[n][3])); }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, x)); }
      const float na = fmaxf(ma, xa * a.scale_log2), nb = fmaxf(mb, xb * a.scale_log2);
      const float ua = na == -INFINITY ? 0.f : na, ub = nb == -INFINITY ? 0.f : nb;   // nothing seen yet: every exponential is exp(-inf)
      const float fa = exp2f(ma - ua), fb = exp2f(mb - ub);
      ma = na; mb = nb;
      float ta = 0.f, tb = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        p[n][0] = exp2f(fmaf(p[n][0], a.scale_log2, head - ua)); p[n][1] = exp2f(fmaf(p[n][1], a.scale_log2, head - ua));
        p[n][2] = exp2f(fmaf(p[n][2], a.scale_log2, head - ub)); p[n][3] = exp2f(fmaf(p[n][3], a.scale_log2, head - ub));
        ta += p[n][0] + p[n][1]; tb += p[n][2] + p[n][3];
      }
      la = fmaf(la, fa, ta); lb = fmaf(lb, fb, tb);
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) { o[n][0] *= fa; o[n][1] *= fa; o[n][2] *= fb; o[n][3] *= fb; }
      product_nn<T, DP, NT>(o, p, sv + buf * BN * L::kStride, lane, cols);
    }
    __syncthreads();
  }
  copy_wait<0>();
  if (wr >= rows) return;
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) { la += __shfl_xor_sync(0xffffffffu, la, x); lb += __shfl_xor_sync(0xffffffffu, lb, x); }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int pr = half ? rb : ra;
    if (pr >= rows) continue;
    const float m = (half ? mb : ma) - head, l = half ? lb : la;
    if (SPLIT && item.y > 1) {
      const size_t slot = ((size_t)unit * a.hk + hy) * a.part_rows + pr;
      float* dst = a.part_o + slot * DP + 2 * (lane & 3);
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
      if ((lane & 3) == 0) a.part_ml[slot] = make_float2(m, l);
      continue;
    }
    const int tok = SPLIT ? pr / G : pr, head = SPLIT ? hy * G + pr % G : hy;
    if (!SPLIT && a.pieces > 1) {
      const long long slot = ((long long)piece * a.hq + head) * a.nq + q0 + tok;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        const int c = n * 8 + 2 * (lane & 3);
        if (c < a.d) *reinterpret_cast<float2*>(a.part_o + slot * a.d + c) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
      }
      if ((lane & 3) == 0) a.part_ml[slot] = make_float2(m, l);
      continue;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);               // a row without keys gives zero; NaN stays NaN
    const long long to = ((long long)(q0 + tok) * a.hq + head) * a.d;
    T *dst = static_cast<T*>(a.out) + to, *rest = a.out_rest ? static_cast<T*>(a.out_rest) + to : nullptr;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      const int c = n * 8 + 2 * (lane & 3);
      if (c < a.d) store_rest<T>(dst + c, rest ? rest + c : nullptr, o[n][2 * half] * inv, o[n][2 * half + 1] * inv);
    }
    if ((lane & 3) == 0 && a.lse) a.lse[(long long)head * a.nq + q0 + tok] = l == 0.f ? -INFINITY : m + log2f(l);
  }
}

// The split form for up to 16 rows (a new token of a few heads): bound by the keys and values that go by, so every warp streams its own 16 of
// 64 keys through buffers of its own, without a barrier of the CTA, and the four partial results meet at the end.
constexpr int kNarrowRows = 16;
template <typename T, int DP> constexpr int narrow_stages() { return sizeof(T) == 4 && DP > 64 ? 2 : 3; }
template <typename T, int DP> constexpr int narrow_smem() { return (kNarrowRows + 4 * narrow_stages<T, DP>() * 32) * Tile<T, DP>::kStride; }
template <typename T, int DP>
__global__ void __launch_bounds__(128) narrow_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int ST = narrow_stages<T, DP>();
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sq = smem_addr(smem), sk = sq + (kNarrowRows + warp * ST * 32) * L::kStride;      // stages of 16 keys, then 16 values
  const int4 item = a.items[blockIdx.x / a.hk];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int G = a.group, hy = blockIdx.x % a.hk, rows = lq * G, k0 = item.z + warp * 16, k1 = item.w;
  const int nt = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;
  const T *kp = static_cast<const T*>(a.k.p) + hy * a.k.head, *vp = static_cast<const T*>(a.v.p) + hy * a.v.head;
  auto load = [&](int it) {
    if (it < nt) {
      const uint32_t at = sk + (it % ST) * 32 * L::kStride;
      const int b = k0 + it * 64;
#pragma unroll
      for (int i = lane; i < 16 * L::kChunks; i += 32) {
        const int r = i / L::kChunks, c = i % L::kChunks;
        const bool ok = b + r < k1 && c * L::kPer < a.d;
        copy16(at + r * L::kStride + c * 16, ok ? kp + (long long)(c0 + b + r) * a.k.row + c * L::kPer : kp, ok);
        copy16(at + (16 + r) * L::kStride + c * 16, ok ? vp + (long long)(c0 + b + r) * a.v.row + c * L::kPer : vp, ok);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int it = 0; it < ST - 1; ++it) load(it);
  {  // queries, with the first group of every warp's copies waited for below
    const T* p = static_cast<const T*>(a.q.p);
    for (int i = tid; i < kNarrowRows * L::kChunks; i += 128) {
      const int r = i / L::kChunks, c = i % L::kChunks;
      const bool ok = r < rows && c * L::kPer < a.d;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (ok) v = *reinterpret_cast<const uint4*>(p + (long long)(q0 + r / G) * a.q.row + (hy * G + r % G) * a.q.head + c * L::kPer);
      *reinterpret_cast<uint4*>(smem + r * L::kStride + c * 16) = v;
    }
  }
  __syncthreads();
  const int ra = lane >> 2, rb = ra + 8, off = lk - lq, big = 0x7fffffff;
  const int lim_a = a.causal ? ra / G + off : big, lim_b = a.causal ? rb / G + off : big, lim_lo = a.causal ? off : big;
  float o[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
  constexpr float head = kHead<T, false>;
  for (int it = 0; it < nt; ++it) {
    load(it + ST - 1);
    copy_wait<ST - 1>();
    __syncwarp();
    const int kb = k0 + it * 64;
    const uint32_t at = sk + (it % ST) * 32 * L::kStride;
    float p[2][4];
    product_nt<T, DP, 2>(p, sq, at, lane, 16);
    if (kb + 16 > k1 || kb + 15 > lim_lo) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = kb + n * 8 + 2 * (lane & 3) + e;
          if (j >= k1 || j > lim_a) p[n][e] = -INFINITY;
          if (j >= k1 || j > lim_b) p[n][2 + e] = -INFINITY;
        }
      }
    }
    float xa = fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[1][0], p[1][1])), xb = fmaxf(fmaxf(p[0][2], p[0][3]), fmaxf(p[1][2], p[1][3]));
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, x)); }
    const float na = fmaxf(ma, xa * a.scale_log2), nb = fmaxf(mb, xb * a.scale_log2);
    const float ua = na == -INFINITY ? 0.f : na, ub = nb == -INFINITY ? 0.f : nb;
    const float fa = exp2f(ma - ua), fb = exp2f(mb - ub);
    ma = na; mb = nb;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      p[n][0] = exp2f(fmaf(p[n][0], a.scale_log2, head - ua)); p[n][1] = exp2f(fmaf(p[n][1], a.scale_log2, head - ua));
      p[n][2] = exp2f(fmaf(p[n][2], a.scale_log2, head - ub)); p[n][3] = exp2f(fmaf(p[n][3], a.scale_log2, head - ub));
    }
    la = fmaf(la, fa, p[0][0] + p[0][1] + p[1][0] + p[1][1]);
    lb = fmaf(lb, fb, p[0][2] + p[0][3] + p[1][2] + p[1][3]);
    if (__any_sync(0xffffffffu, fa != 1.f || fb != 1.f)) {
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) { o[n][0] *= fa; o[n][1] *= fa; o[n][2] *= fb; o[n][3] *= fb; }
    }
    product_nn<T, DP, 2>(o, p, at + 16 * L::kStride, lane, 16);
    __syncwarp();
  }
  copy_wait<0>();
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) { la += __shfl_xor_sync(0xffffffffu, la, x); lb += __shfl_xor_sync(0xffffffffu, lb, x); }
  // the four warps' shares: (m, l) and o of every row in shared memory, over the buffers
  __syncthreads();
  float* so = reinterpret_cast<float*>(smem);                       // [4][16][DP + 2]
  constexpr int W = DP + 2;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float* dst = so + (warp * kNarrowRows + (half ? rb : ra)) * W;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8 + 2 * (lane & 3)) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
    if ((lane & 3) == 0) *reinterpret_cast<float2*>(dst + DP) = make_float2(half ? mb : ma, half ? lb : la);
  }
  __syncthreads();
  for (int r = warp; r < rows; r += 4) {
    float m = -INFINITY, l = 0.f, f[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, so[(w * kNarrowRows + r) * W + DP]);
    const float u = m == -INFINITY ? 0.f : m;
    m -= head;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = exp2f(so[(w * kNarrowRows + r) * W + DP] - u);
      l = fmaf(so[(w * kNarrowRows + r) * W + DP + 1], f[w], l);
    }
    const size_t slot = ((size_t)(blockIdx.x / a.hk) * a.hk + hy) * a.part_rows + r;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const long long to = ((long long)(q0 + r / G) * a.hq + hy * G + r % G) * a.d;
#pragma unroll
    for (int c = lane; c < DP; c += 32) {
      float x = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) x = fmaf(so[(w * kNarrowRows + r) * W + c], f[w], x);
      if (item.y > 1) {
        a.part_o[slot * DP + c] = x;
      } else if (c < a.d) {
        x *= inv;
        const T y = (T)x;
        static_cast<T*>(a.out)[to + c] = y;
        if (sizeof(T) == 2 && a.out_rest) static_cast<T*>(a.out_rest)[to + c] = (T)(x - (float)y);
      }
    }
    if (lane == 0) {
      if (item.y > 1) a.part_ml[slot] = make_float2(m, l);
      else if (a.lse) a.lse[(long long)(hy * G + r % G) * a.nq + q0 + r / G] = l == 0.f ? -INFINITY : m + log2f(l);
    }
  }
}

// joins the stretches of a structure's keys: a warp per row of the split form
template <typename T, int DP>
__global__ void __launch_bounds__(256) combine_kernel(const PackedArgs a) {
  const int s = blockIdx.x / a.hk, hy = blockIdx.x % a.hk, lane = threadIdx.x & 31;
  const int first = a.split_first[s], n = a.split_first[s + 1] - first;
  const int q0 = a.start_q[s], rows = (a.start_q[s + 1] - q0) * a.group;
  if (n <= 1) return;
  for (int pr = threadIdx.x >> 5; pr < rows; pr += 8) {
    float m = -INFINITY;
    for (int i = lane; i < n; i += 32) m = fmaxf(m, a.part_ml[((size_t)(first + i) * a.hk + hy) * a.part_rows + pr].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    const float u = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[DP / 32];
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) o[c] = 0.f;
    for (int i = 0; i < n; ++i) {
      const size_t slot = ((size_t)(first + i) * a.hk + hy) * a.part_rows + pr;
      const float2 ml = a.part_ml[slot];
      const float f = exp2f(ml.x - u);
      l = fmaf(ml.y, f, l);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) o[c] = fmaf(a.part_o[slot * DP + c * 32 + lane], f, o[c]);
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    const int tok = pr / a.group, head = hy * a.group + pr % a.group;
    const long long to = ((long long)(q0 + tok) * a.hq + head) * a.d;
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
      if (c * 32 + lane >= a.d) continue;
      const float x = o[c] * inv;
      const T y = (T)x;
      static_cast<T*>(a.out)[to + c * 32 + lane] = y;
      if (sizeof(T) == 2 && a.out_rest) static_cast<T*>(a.out_rest)[to + c * 32 + lane] = (T)(x - (float)y);
    }
    if (lane == 0 && a.lse) a.lse[(long long)head * a.nq + q0 + tok] = l == 0.f ? -INFINITY : m + log2f(l);
  }
}

// ---- pieces ----
// joins the pieces of the forward kernel: a thread per eight values of a row
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const PackedArgs a, int rows) {
  const int parts = a.d / 8;
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x, hr = e / parts;
  const int c = (int)(e % parts) * 8;
  if (hr >= (long long)rows * a.hq) return;
  const long long r = hr / a.hq;
  const int h = (int)(hr % a.hq);
  float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  for (int p = 0; p < a.pieces; ++p) m = fmaxf(m, a.part_ml[((long long)p * a.hq + h) * a.nq + r].x);
  const float u = m == -INFINITY ? 0.f : m;
  for (int p = 0; p < a.pieces; ++p) {
    const long long slot = ((long long)p * a.hq + h) * a.nq + r;
    const float2 ml = a.part_ml[slot];
    if (ml.y == 0.f) continue;      // no key of the piece was seen: its share was not written where it has no tile
    const float f = exp2f(ml.x - u);
    l = fmaf(ml.y, f, l);
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + slot * a.d + c), y = *reinterpret_cast<const float4*>(a.part_o + slot * a.d + c + 4);
    o[0] = fmaf(x.x, f, o[0]); o[1] = fmaf(x.y, f, o[1]); o[2] = fmaf(x.z, f, o[2]); o[3] = fmaf(x.w, f, o[3]);
    o[4] = fmaf(y.x, f, o[4]); o[5] = fmaf(y.y, f, o[5]); o[6] = fmaf(y.z, f, o[6]); o[7] = fmaf(y.w, f, o[7]);
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  const long long at = hr * a.d + c;
#pragma unroll
  for (int k = 0; k < 8; k += 2) store_rest<T>(static_cast<T*>(a.out) + at + k, a.out_rest ? static_cast<T*>(a.out_rest) + at + k : nullptr, o[k] * inv, o[k + 1] * inv);
  if (c == 0 && a.lse) a.lse[(long long)h * a.nq + r] = l == 0.f ? -INFINITY : m + log2f(l);
}
// sums the pieces' shares of dq, dk, dv (blockIdx.y), a thread per eight values
template <typename T>
__global__ void __launch_bounds__(256) sum_kernel(const PackedArgs a, int first, int pieces_q, int pieces_kv, long long values_q, long long values_kv,
                                                  long long stride_q, long long stride_kv) {
  const int which = first + blockIdx.y, pieces = which ? pieces_kv : pieces_q;
  const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * 8, values = which ? values_kv : values_q, stride = which ? stride_kv : stride_q;
  if (e >= values) return;
  const float* src = a.share[which] + e;
  float o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) o[k] = 0.f;
  for (int p = 0; p < pieces; ++p) {
    const float4 x = *reinterpret_cast<const float4*>(src + p * stride), y = *reinterpret_cast<const float4*>(src + p * stride + 4);
    o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w; o[4] += y.x; o[5] += y.y; o[6] += y.z; o[7] += y.w;
  }
  T* dst = static_cast<T*>(which == 0 ? a.dq : which == 1 ? a.dk : a.dv) + e;
#pragma unroll
  for (int k = 0; k < 8; k += 2) store2(dst + k, o[k], o[k + 1]);
}

// ---- reverse --------------------------------------------------------------------------------------------------------
// g . o of 16 bytes with what rounding o left, and g . g of a 16-bit type
template <typename T>
__device__ __forceinline__ void dot16(const uint4 g, const uint4 o, const uint4 rest, float& sum, float& square) {
  const uint32_t xs[4] = {g.x, g.y, g.z, g.w}, ys[4] = {o.x, o.y, o.z, o.w}, zs[4] = {rest.x, rest.y, rest.z, rest.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (sizeof(T) == 2) {
      const float2 u = Half<T>::unpack(xs[e]), v = Half<T>::unpack(ys[e]), w = Half<T>::unpack(zs[e]);
      sum = fmaf(u.x, v.x + w.x, fmaf(u.y, v.y + w.y, sum));
      square = fmaf(u.x, u.x, fmaf(u.y, u.y, square));
    } else {
      sum = fmaf(__uint_as_float(xs[e]), __uint_as_float(ys[e]), sum);
    }
  }
}
template <typename T> __device__ __forceinline__ uint4 load16(const void* p, long long at) { return *reinterpret_cast<const uint4*>(static_cast<const T*>(p) + at); }
// delta = sum over d of g * o, a thread per 16 bytes, rows of all heads; empties the queues of the kernels behind it
template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(const PackedArgs a, int rows, int width) {
  constexpr int V = 16 / (int)sizeof(T);
  if (a.queue && blockIdx.x == 0 && threadIdx.x < 2) a.queue[threadIdx.x] = 0;
  const int part = threadIdx.x % width;
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) / width;
  const long long r = i / a.hq;
  const int h = (int)(i % a.hq);
  float sum = 0.f, square = 0.f;
  if (r < rows && part * V < a.d) {
    const long long at = (r * a.hq + h) * a.d + part * V;
    dot16<T>(load16<T>(a.g.p, r * a.g.row + h * a.g.head + part * V), load16<T>(a.o.p, at),
             sizeof(T) == 2 && a.out_rest ? load16<T>(a.out_rest, at) : make_uint4(0, 0, 0, 0), sum, square);
  }
  for (int x = width >> 1; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
  if (r < rows && part == 0) a.delta[(long long)h * a.nq + r] = sum;
}
// The same with the sizes of g and v (PackedArgs::largest, size_g), for the tensor-core kernels of float16: a CTA per 128 / parts rows of a tile of 128
// queries and up to 64 heads, and behind these CTAs for the keys.  A warp takes two rows of 32 / width heads at a time, so that no thread divides
// and a head's largest stays in a register.  The order of the atomics, one a CTA and head, does not matter.  |v| is bounded by sqrt(d) times
// its largest value, which needs no sum.  (24 structures of 150 to 900 rows, 16 heads x 64: 26 us, where delta alone takes 16.)
constexpr int kSizeHeads = 64;
template <typename T>
__global__ void __launch_bounds__(256) delta_sizes_kernel(const PackedArgs a, const int4* items_q, long long ctas_q, const int4* items_kv, int log_width, int parts) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ unsigned most[kSizeHeads];
  if (a.queue && blockIdx.x == 0 && threadIdx.x < 2) a.queue[threadIdx.x] = 0;
  const bool of_v = blockIdx.x >= ctas_q;
  const int all = of_v ? a.hk : a.hq, blocks = (all + kSizeHeads - 1) / kSizeHeads, index = (int)(blockIdx.x - (of_v ? ctas_q : 0));
  const int4 item = (of_v ? items_kv : items_q)[index / parts / blocks];
  const int* start = of_v ? a.start_kv : a.start_q;
  const int per = 128 / parts, row0 = item.y * 128 + index % parts * per, first = start[item.x] + row0, rows = min(per, start[item.x + 1] - first);
  if (rows <= 0) return;
  const int h0 = index / parts % blocks * kSizeHeads, heads = min(kSizeHeads, all - h0), width = 1 << log_width;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = lane & (width - 1);
  if (threadIdx.x < kSizeHeads) most[threadIdx.x] = 0;
  __syncthreads();
  const bool on = part * V < a.d;
  for (int hb = 0; hb < heads; hb += 32 >> log_width) {      // the same trips for all lanes
    const int hh = hb + (lane >> log_width), h = h0 + hh;
    float size = 0.f;
    for (int row = warp; row < rows + warp; row += 16) {
      uint4 g[2], o[2], rest[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const long long r = first + row + 8 * u;
        g[u] = o[u] = rest[u] = make_uint4(0, 0, 0, 0);
        if (row + 8 * u < rows && hh < heads && on) {
          const Rows& x = of_v ? a.v : a.g;
          g[u] = load16<T>(x.p, r * x.row + h * x.head + part * V);
          if (!of_v) {
            const long long at = (r * a.hq + h) * a.d + part * V;
            o[u] = load16<T>(a.o.p, at);
            if (a.out_rest) rest[u] = load16<T>(a.out_rest, at);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // one that is not finite spoils its rows whatever their power of two: left out
        if (of_v) {
          const uint32_t xs[4] = {g[u].x, g[u].y, g[u].z, g[u].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x = Half<T>::unpack(xs[e]);
            if (isfinite(x.x)) size = fmaxf(size, fabsf(x.x));
            if (isfinite(x.y)) size = fmaxf(size, fabsf(x.y));
          }
        } else {
          float sum = 0.f, square = 0.f;
          dot16<T>(g[u], o[u], rest[u], sum, square);
          for (int x = width >> 1; x; x >>= 1) { sum += __shfl_xor_sync(0xffffffffu, sum, x); square += __shfl_xor_sync(0xffffffffu, square, x); }
          const float norm = sqrtf(square);
          if (row + 8 * u < rows && hh < heads && part == 0) {
            const long long at = (long long)h * a.nq + first + row + 8 * u;
            a.delta[at] = sum;
            a.size_g[at] = norm;
          }
          if (isfinite(norm)) size = fmaxf(size, norm);
        }
      }
    }
    if (of_v) {
      for (int x = width >> 1; x; x >>= 1) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, x));
      size *= sqrtf((float)a.d);
    }
    if (hh < heads && part == 0) atomicMax(&most[hh], __float_as_uint(size));      // not negative: ordered as their bits are
  }
  __syncthreads();
  if (threadIdx.x < heads) atomicMax(a.largest + ((long long)item.x * a.hk + (h0 + threadIdx.x) / (of_v ? 1 : a.group)) * 2 + of_v, most[threadIdx.x]);
}

// float16: the power of two of dS (grad_shift) from the values themselves, of every row of the product.  A row's first value that is not zero sets it, and
// it falls where a value would pass 2^15; what was summed so far is scaled along, exactly.  `v`: rows a and b of this thread, shared by four
// lanes, times the present powers.  Not above 2^80, with which float32 holds any |dS| of float16 rows (2^39).  (With sizes found ahead as for
// the tensor cores: 512 structures of 10 to 40, 4 x 32, 48 us a training step instead of 35, 50,000 of two rows 2,550 instead of 1,240.)
struct RowShift {
  int shift = 0;
  float top = 0.f;
};
template <int NT, int DP> __device__ __forceinline__ void shift_rows(float (&v)[NT][4], float (&acc)[DP / 8][4], RowShift& a, RowShift& b) {
  float xa = 0.f, xb = 0.f;
#pragma unroll
  for (int n = 0; n < NT; ++n) { xa = fmaxf(xa, fmaxf(fabsf(v[n][0]), fabsf(v[n][1]))); xb = fmaxf(xb, fmaxf(fabsf(v[n][2]), fabsf(v[n][3]))); }
  if (!__any_sync(0xffffffffu, xa > a.top || xb > b.top)) return;
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) { xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, x)); xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, x)); }
  auto factor = [](float x, RowShift& r) {
    if (!(x > r.top)) return 1.f;
    const int by = min(14 - ((int)(__float_as_uint(x) >> 23) - 127), 80 - r.shift);
    r.shift += by; r.top = 32768.f;
    return two_to(max(by, -126));
  };
  const float fa = factor(xa, a), fb = factor(xb, b);
#pragma unroll
  for (int n = 0; n < NT; ++n) { v[n][0] *= fa; v[n][1] *= fa; v[n][2] *= fb; v[n][3] *= fb; }
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) { acc[n][0] *= fa; acc[n][1] *= fa; acc[n][2] *= fb; acc[n][3] *= fb; }
}

// dq of a tile of 16 NW queries of one head
template <typename T, int DP, int NW>
__global__ void __launch_bounds__(32 * NW) dq_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int BN = kRevTile, NT = BN / 8, kRows = 16 * NW, kThreads = 32 * NW;
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sq = smem_addr(smem), sg = sq + kRows * L::kStride, sk = sg + kRows * L::kStride, sv = sk + a.rev_stages * BN * L::kStride;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int piece = blockIdx.x % a.pieces, index = blockIdx.x / a.pieces;
  const int4 item = a.items[index / a.hq];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int h = index % a.hq, kvh = h / a.group, row0 = item.y * kRows;
  const int share = ((item.w + BN - 1) / BN + a.pieces - 1) / a.pieces * BN, k0 = min(item.w, piece * share), k1 = min(item.w, k0 + share);
  const int nt = (max(k1 - k0, 0) + BN - 1) / BN;
  load_rows<T, DP, kRows, kThreads>(sq, a.q, h, q0, row0, lq, a.d, tid);
  load_rows<T, DP, kRows, kThreads>(sg, a.g, h, q0, row0, lq, a.d, tid);
  auto load = [&](int it) {
    if (it < nt) {
      const int buf = it & (a.rev_stages - 1), b = k0 + it * BN;
      load_rows<T, DP, BN, kThreads>(sk + buf * BN * L::kStride, a.k, kvh, c0, b, k1, a.d, tid);
      load_rows<T, DP, BN, kThreads>(sv + buf * BN * L::kStride, a.v, kvh, c0, b, k1, a.d, tid);
    }
    copy_commit();
  };
  load(0);
  const int wr = row0 + warp * 16, ra = wr + (lane >> 2), rb = ra + 8, off = lk - lq, big = 0x7fffffff;
  const int lim_a = a.causal ? ra + off : big, lim_b = a.causal ? rb + off : big, lim_lo = a.causal ? wr + off : big, lim_hi = a.causal ? wr + 15 + off : big;
  const long long at_row = (long long)h * a.nq + q0;
  // rows that are not there: exp(-inf) = 0
  const float ea = ra < lq ? a.lse[at_row + ra] : INFINITY, eb = rb < lq ? a.lse[at_row + rb] : INFINITY;
  const float da = ra < lq ? a.delta[at_row + ra] : 0.f, db = rb < lq ? a.delta[at_row + rb] : 0.f;
  float dq[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) dq[n][0] = dq[n][1] = dq[n][2] = dq[n][3] = 0.f;
  RowShift sh_a, sh_b;      // of the rows' dS and what was summed of them
  for (int it = 0; it < nt; ++it) {
    if (a.rev_stages == 2) { load(it + 1); copy_wait<1>(); } else { if (it > 0) load(it); copy_wait<0>(); }
    __syncthreads();
    const int kb = k0 + it * BN, buf = it & (a.rev_stages - 1);
    if (wr < lq && kb <= lim_hi) {
      float p[NT][4], dp[NT][4];
      const int cols = k1 - kb;
      product_nt<T, DP, NT>(p, sq + warp * 16 * L::kStride, sk + buf * BN * L::kStride, lane, cols);
      product_nt<T, DP, NT>(dp, sg + warp * 16 * L::kStride, sv + buf * BN * L::kStride, lane, cols);
      const bool mask = kb + BN > k1 || kb + BN - 1 > lim_lo;
      const float ua = kShifted<T> ? sh_a.shift - ea : -ea, ub = kShifted<T> ? sh_b.shift - eb : -eb;      // P times the power of dS
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = kb + n * 8 + 2 * (lane & 3) + e;
          float x = exp2f(fmaf(p[n][e], a.scale_log2, ua)) * (dp[n][e] - da);
          float y = exp2f(fmaf(p[n][2 + e], a.scale_log2, ub)) * (dp[n][2 + e] - db);
          if (mask && (j >= k1 || j > lim_a)) x = 0.f;
          if (mask && (j >= k1 || j > lim_b)) y = 0.f;
          p[n][e] = x; p[n][2 + e] = y;
        }
      }
      if constexpr (kShifted<T>) shift_rows<NT, DP>(p, dq, sh_a, sh_b);
      product_nn<T, DP, NT>(dq, p, sk + buf * BN * L::kStride, lane, cols);
    }
    __syncthreads();
  }
  copy_wait<0>();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half ? rb : ra;
    if (r >= lq) continue;
    const long long at = ((long long)(q0 + r) * a.hq + h) * a.d;
    const float f = kShifted<T> ? a.scale * two_to(-(half ? sh_b.shift : sh_a.shift)) : a.scale;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      const int c = n * 8 + 2 * (lane & 3);
      if (c >= a.d) continue;
      const float x = dq[n][2 * half] * f, y = dq[n][2 * half + 1] * f;
      if (a.pieces > 1) store2(a.share[0] + (long long)piece * a.nq * a.hq * a.d + at + c, x, y);
      else store2(static_cast<T*>(a.dq) + at + c, x, y);
    }
  }
}

// dk and dv of a tile of 16 NW keys of one key head: rows of the products are keys, columns queries
template <typename T, int DP, int NW>
__global__ void __launch_bounds__(32 * NW) dkv_kernel(const PackedArgs a) {
  using L = Tile<T, DP>;
  constexpr int BN = kRevTile, NT = BN / 8, kRows = 16 * NW, kThreads = 32 * NW;
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t sk = smem_addr(smem), sv = sk + kRows * L::kStride, sq = sv + kRows * L::kStride, sg = sq + a.rev_stages * BN * L::kStride;
  float* se = reinterpret_cast<float*>(smem + (2 * kRows + 2 * a.rev_stages * BN) * L::kStride);   // [2][BN] lse, [2][BN] delta
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int piece = blockIdx.x % a.pieces, index = blockIdx.x / a.pieces;
  const int4 item = a.items[index / a.hk];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int kvh = index % a.hk, row0 = item.y * kRows, i0 = item.z, i1 = item.w;
  const int per = (max(i1 - i0, 0) + BN - 1) / BN, all = per * a.group, share = (all + a.pieces - 1) / a.pieces, j0 = min(all, piece * share);
  const int nt = min(share, all - j0);      // from tile j0 on
  load_rows<T, DP, kRows, kThreads>(sk, a.k, kvh, c0, row0, lk, a.d, tid);
  load_rows<T, DP, kRows, kThreads>(sv, a.v, kvh, c0, row0, lk, a.d, tid);
  auto load = [&](int it) {
    if (it < nt) {
      const int buf = it & (a.rev_stages - 1), h = kvh * a.group + (j0 + it) / per, b = i0 + ((j0 + it) % per) * BN;
      load_rows<T, DP, BN, kThreads>(sq + buf * BN * L::kStride, a.q, h, q0, b, i1, a.d, tid);
      load_rows<T, DP, BN, kThreads>(sg + buf * BN * L::kStride, a.g, h, q0, b, i1, a.d, tid);
      if (tid < BN) {
        const bool ok = b + tid < i1;
        const long long at = (long long)h * a.nq + q0 + b + tid;
        se[buf * BN + tid] = ok ? a.lse[at] - prob_shift<T>() : INFINITY;
        se[(2 + buf) * BN + tid] = ok ? a.delta[at] * prob_unscale<T>() : 0.f;
      }
    }
    copy_commit();
  };
  load(0);
  const int wr = row0 + warp * 16, ra = wr + (lane >> 2), rb = ra + 8, off = lk - lq, none = -0x7fffffff - 1;
  // first query that sees a key
  const int lim_a = a.causal ? ra - off : none, lim_b = a.causal ? rb - off : none, lim_lo = a.causal ? wr - off : none, lim_hi = a.causal ? wr + 15 - off : none;
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) { dk[n][0] = dk[n][1] = dk[n][2] = dk[n][3] = 0.f; dv[n][0] = dv[n][1] = dv[n][2] = dv[n][3] = 0.f; }
  RowShift sh_a, sh_b;
  for (int it = 0; it < nt; ++it) {
    if (a.rev_stages == 2) { load(it + 1); copy_wait<1>(); } else { if (it > 0) load(it); copy_wait<0>(); }
    __syncthreads();
    const int ib = i0 + ((j0 + it) % per) * BN, buf = it & (a.rev_stages - 1);
    if (wr < lk && ib + BN - 1 >= lim_lo) {
      float p[NT][4], ds[NT][4];
      const int cols = i1 - ib;
      product_nt<T, DP, NT>(p, sk + warp * 16 * L::kStride, sq + buf * BN * L::kStride, lane, cols);
      product_nt<T, DP, NT>(ds, sv + warp * 16 * L::kStride, sg + buf * BN * L::kStride, lane, cols);
      const bool mask = a.causal && ib < lim_hi;
      const float pa = kShifted<T> ? two_to(sh_a.shift) : 1.f, pb = kShifted<T> ? two_to(sh_b.shift) : 1.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int c = n * 8 + 2 * (lane & 3);
        const float2 e = *reinterpret_cast<const float2*>(se + buf * BN + c), d = *reinterpret_cast<const float2*>(se + (2 + buf) * BN + c);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = ib + c + (x & 1), lim = x < 2 ? lim_a : lim_b;
          float w = exp2f(fmaf(p[n][x], a.scale_log2, -((x & 1) ? e.y : e.x)));
          if (mask && i < lim) w = 0.f;
          ds[n][x] = w == 0.f ? 0.f : w * fmaf(ds[n][x], prob_unscale<T>(), -((x & 1) ? d.y : d.x)) * (x < 2 ? pa : pb);
          p[n][x] = w;
        }
      }
      product_nn<T, DP, NT>(dv, p, sg + buf * BN * L::kStride, lane, cols);
      if constexpr (kShifted<T>) shift_rows<NT, DP>(ds, dk, sh_a, sh_b);
      product_nn<T, DP, NT>(dk, ds, sq + buf * BN * L::kStride, lane, cols);
    }
    __syncthreads();
  }
  copy_wait<0>();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = half ? rb : ra;
    if (r >= lk) continue;
    const float f = kShifted<T> ? a.scale * two_to(-(half ? sh_b.shift : sh_a.shift)) : a.scale;
    const long long at = ((long long)(c0 + r) * a.hk + kvh) * a.d;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      const int c = n * 8 + 2 * (lane & 3);
      if (c >= a.d) continue;
      const float k0 = dk[n][2 * half] * f, k1 = dk[n][2 * half + 1] * f;
      const float v0 = dv[n][2 * half] * prob_unscale<T>(), v1 = dv[n][2 * half + 1] * prob_unscale<T>();
      if (a.pieces > 1) {
        const long long to = (long long)piece * a.nkv * a.hk * a.d + at + c;
        store2(a.share[1] + to, k0, k1);
        store2(a.share[2] + to, v0, v1);
      } else {
        store2(static_cast<T*>(a.dk) + at + c, k0, k1);
        store2(static_cast<T*>(a.dv) + at + c, v0, v1);
      }
    }
  }
}

// The attribute holds per device for good: set once (a repeated call costs a microsecond).  A lost race sets it twice.
template <auto kernel>
void allow_smem(int smem) {
  static std::atomic<int> most[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64 || most[dev].load(std::memory_order_acquire) < smem) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess && dev < 64) most[dev].store(smem, std::memory_order_release);
  }
}
template <auto kernel>
int launch(int64_t grid, int threads, int smem, cudaStream_t st, const PackedArgs& a) {
  if (grid > 0x7fffffff) return kTooLarge;
  if (smem > 48 * 1024) allow_smem<kernel>(smem);
  kernel<<<(unsigned)grid, threads, smem, st>>>(a);
  count_launch();
  return kOk;
}

#define SO3LR_PACKED_WIDTHS(T, CALL)            \
  switch (packed_padded(a.d)) {                 \
    case 32: { CALL(T, 32) }                    \
    case 64: { CALL(T, 64) }                    \
    case 96: { CALL(T, 96) }                    \
    default: { CALL(T, 128) }                   \
  }

}  // namespace packed

template <typename T> int packed_forward_mma(cudaStream_t st, const PackedArgs& a, int n_items) {
  const int64_t grid = (int64_t)n_items * a.hq * a.pieces;
#define CALL(T, DP)                                                                                                                             \
  return a.tile_rows == 16 ? packed::launch<packed::forward_kernel<T, DP, false, 1>>(grid, 32, packed::forward_smem<T, DP, 1>(a.stages), st, a) \
                           : packed::launch<packed::forward_kernel<T, DP, false, 4>>(grid, 128, packed::forward_smem<T, DP, 4>(a.stages), st, a);
  SO3LR_PACKED_WIDTHS(T, CALL)
#undef CALL
}
template <typename T> int packed_forward_split(cudaStream_t st, const PackedArgs& a, int n_items, int n_structures, bool combine) {
  const int64_t grid = (int64_t)n_items * a.hk;
#define CALL(T, DP)                                                                                                                             \
  const int rc = a.part_rows <= packed::kNarrowRows                                                                                             \
                     ? packed::launch<packed::narrow_kernel<T, DP>>(grid, 128, packed::narrow_smem<T, DP>(), st, a)                             \
                     : packed::launch<packed::forward_kernel<T, DP, true, 4>>(grid, 128, packed::forward_smem<T, DP, 4>(a.stages), st, a);      \
  return rc || !combine ? rc : packed::launch<packed::combine_kernel<T, DP>>((int64_t)n_structures * a.hk, 256, 0, st, a);
  SO3LR_PACKED_WIDTHS(T, CALL)
#undef CALL
}
template <typename T> int packed_dq_mma(cudaStream_t st, const PackedArgs& a, int n_items) {
  const int64_t grid = (int64_t)n_items * a.hq * a.pieces;
#define CALL(T, DP)                                                                                                                        \
  return a.tile_rows == 16 ? packed::launch<packed::dq_kernel<T, DP, 1>>(grid, 32, packed::reverse_smem<T, DP, 1>(a.rev_stages), st, a)    \
                           : packed::launch<packed::dq_kernel<T, DP, 4>>(grid, 128, packed::reverse_smem<T, DP, 4>(a.rev_stages), st, a);
  SO3LR_PACKED_WIDTHS(T, CALL)
#undef CALL
}
template <typename T> int packed_dkv_mma(cudaStream_t st, const PackedArgs& a, int n_items) {
  const int64_t grid = (int64_t)n_items * a.hk * a.pieces;
#define CALL(T, DP)                                                                                                                        \
  return a.tile_rows == 16 ? packed::launch<packed::dkv_kernel<T, DP, 1>>(grid, 32, packed::reverse_smem<T, DP, 1>(a.rev_stages), st, a)   \
                           : packed::launch<packed::dkv_kernel<T, DP, 4>>(grid, 128, packed::reverse_smem<T, DP, 4>(a.rev_stages), st, a);
  SO3LR_PACKED_WIDTHS(T, CALL)
#undef CALL
}
template <typename T> int packed_join(cudaStream_t st, const PackedArgs& a) {
  const int64_t ctas = ((int64_t)a.rows * a.hq * (a.d / 8) + 255) / 256;
  if (ctas > 0x7fffffff) return kTooLarge;
  packed::join_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(a, a.rows);
  count_launch();
  return kOk;
}
template <typename T> int packed_sum(cudaStream_t st, const PackedArgs& a, int pieces_q, int pieces_kv) {
  const long long values_q = (long long)a.rows * a.hq * a.d, values_kv = (long long)a.rows_kv * a.hk * a.d;
  const int first = pieces_q > 1 ? 0 : 1, many = (pieces_kv > 1 ? 3 : 1) - first;
  const long long most = pieces_q > 1 && (pieces_kv == 1 || values_q > values_kv) ? values_q : values_kv;
  const int64_t ctas = (most / 8 + 255) / 256;
  if (ctas > 0x7fffffff) return kTooLarge;
  packed::sum_kernel<T><<<dim3((unsigned)ctas, many), 256, 0, st>>>(a, first, pieces_q, pieces_kv, values_q, values_kv, (long long)a.nq * a.hq * a.d,
                                                                    (long long)a.nkv * a.hk * a.d);
  count_launch();
  return kOk;
}
template <typename T> int packed_delta(cudaStream_t st, const PackedArgs& a, const int4* items_q, int n_q, const int4* items_kv, int n_kv) {
  int width = 1;
  while (width * (16 / (int)sizeof(T)) < a.d) width <<= 1;
  if (a.rows == 0) return kOk;
  if constexpr (kShifted<T>) {
    if (a.largest) {
      auto blocks = [](int heads) { return (int64_t)((heads + packed::kSizeHeads - 1) / packed::kSizeHeads); };
      const int64_t whole = blocks(a.hq) * n_q + blocks(a.hk) * n_kv;
      int parts = 8, log_width = 0;
      while (parts > 1 && whole * parts > 16384) parts >>= 1;      // many structures, most of them short: CTAs without a row cost some 10 ns each
      while (1 << log_width < width) ++log_width;
      if (whole * parts > 0x7fffffff) return kTooLarge;
      SO3LR_CUDA_CHECK(cudaMemsetAsync(a.largest, 0, (size_t)a.structures * a.hk * 2 * sizeof(unsigned), st));
      packed::delta_sizes_kernel<T><<<(unsigned)(whole * parts), 256, 0, st>>>(a, items_q, blocks(a.hq) * n_q * parts, items_kv, log_width, parts);
      count_launch();
      return kOk;
    }
  }
  const int64_t ctas = ((int64_t)a.rows * a.hq * width + 255) / 256;
  if (ctas > 0x7fffffff) return kTooLarge;
  packed::delta_kernel<T><<<(unsigned)ctas, 256, 0, st>>>(a, a.rows, width);
  count_launch();
  return kOk;
}

}  // namespace so3lr
