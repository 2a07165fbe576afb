// Attention inside the structures of a packed batch on the tensor cores (tcgen05) for 16-bit operands: forward and the two halves of the
// reverse pass, for structures long enough to fill tiles of 128 rows.  The mathematics is that of packed_mma.cuh.
//
// A CTA has the SM to itself: eight warps do the softmax (a thread per row, or per row and half of the columns), one warp issues the
// matrix instructions, three load tiles.  Accumulators and P / dS live in tensor memory: P and dS go back there packed to 16 bits over
// the logits they were made from, and are the A operand of the next product, so shared memory carries q, k, v and g only.
#include "packed_tc.cuh"

namespace so3lr {

__device__ int g_packed_error;      // a bounded wait ran out (so3lr_b200_structure_attention_error)

namespace {

using namespace tc;

// barriers and scratch behind the tiles
struct Tail {
  unsigned long long bars[32];
  uint32_t tmem;
  int failed;
};
// Tiles that stream through: a ring of four slots (two sub-tiles) or eight, the two kinds of tile in turn; tile j sits in slot j % R.
__device__ __forceinline__ int ring_slots(int subs) { return subs == 2 ? 4 : 8; }
// sub-tiles need 1024-byte alignment
__device__ __forceinline__ unsigned char* aligned_smem(unsigned char* p) { return p + ((1024u - (smem_addr(p) & 1023u)) & 1023u); }

// ---- forward --------------------------------------------------------------------------------------------------------
// 256 queries of one head: two tiles of 128 rows take turns, so that the exponentials of one run beside the products of the other.
// Tensor memory: logits of tile t at 128 t, its output at 256 + 128 t; P of a tile replaces its logits.
// The running maximum that the exponentials refer to is raised only where it would grow by more than 8 (in log2): P stays below 2^8, and
// the output, which the tensor cores add to, is rescaled a few times per row instead of once per tile of keys.
enum FwdBar { kFull, kEmpty = kFull + 8, kQFull = kEmpty + 8, kSFull = kQFull + 2, kPFull = kSFull + 2, kOFull = kPFull + 2, kFix = kOFull + 2, kFwdBars };

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) forward_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d, subs = d > 64 ? 2 : 1, tile_bytes = subs * kSub, R = ring_slots(subs);
  Tail* tail = reinterpret_cast<Tail*>(smem + (2 + R) * tile_bytes);
  const uint32_t sq = smem_addr(smem), ring = sq + 2 * tile_bytes, bar0 = smem_addr(tail->bars);
  volatile int* failed = &tail->failed;
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 item = a.items[blockIdx.x];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int h = blockIdx.y, kvh = h / a.group, row0 = item.y * 2 * kTile, off = lk - lq;
  // keys that a tile meets: [0, end[t]), and tiles of keys
  const int end1 = item.w, end0 = a.causal ? min(end1, max(0, min(lq, row0 + kTile) + off)) : end1;
  const int n0 = (end0 + kTile - 1) / kTile, n1 = row0 + kTile < lq ? (end1 + kTile - 1) / kTile : 0, n = max(n0, n1);
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kFwdBars; ++i) init_bar(bar(i), i == kPFull || i == kPFull + 1 ? kTile : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;

  if (warp >= kMmaWarp) {
    fewer_regs<kOtherRegs>();
    if (warp == kMmaWarp && n > 0) {
      const uint32_t on = elect_one();
      // keys are tiles 0, 2, .. of the ring, values 1, 3, ..; a slot is given back only where another tile waits for it, so that nothing is
      // pending when the CTA ends
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };
      auto ready = [&](int j) { wait_bar(bar(kFull + j % R), (j / R) & 1, failed, &g_packed_error); };
      auto give = [&](int j) { if (j + R < 2 * n) commit(on, bar(kEmpty + j % R)); };
      ready(0);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if ((t ? n1 : n0) == 0) continue;
        wait_bar(bar(kQFull + t), 0, failed, &g_packed_error);
        fence_after();
        product_rows<T>(on, tmem + kTile * t, sq + t * tile_bytes, slot(0), d);
        commit(on, bar(kSFull + t));
      }
      give(0);
      for (int i = 0; i < n; ++i) {
        ready(2 * i + 1);
        if (i + 1 < n) ready(2 * i + 2);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int nt = t ? n1 : n0;
          if (i >= nt) continue;
          wait_bar(bar(kPFull + t), i & 1, failed, &g_packed_error);
          fence_after();
          product_cols<T>(on, tmem + 256 + kTile * t, tmem + kTile * t, 32, slot(2 * i + 1), d, i > 0);
          if (i + 1 < nt) {
            product_rows<T>(on, tmem + kTile * t, sq + t * tile_bytes, slot(2 * i + 2), d);
            commit(on, bar(kSFull + t));
          } else {
            commit(on, bar(kOFull + t));
          }
        }
        give(2 * i + 1);
        if (i + 1 < n) give(2 * i + 2);
      }
    } else if (warp == kLoadWarp && n > 0) {
      Loader ld{lane, subs, bar(kFix)};
      for (int t = 0; t < 2; ++t)
        if ((t ? n1 : n0) > 0) ld.tile(sq + t * tile_bytes, &maps.q, q0 + row0 + t * kTile, h, bar(kQFull + t), kTile, false, failed, &g_packed_error);
      for (int j = 0; j < 2 * n; ++j) {
        if (j >= R) wait_bar(bar(kEmpty + j % R), (j / R - 1) & 1, failed, &g_packed_error);
        const int r = (j >> 1) * kTile;
        ld.tile(ring + (j % R) * tile_bytes, (j & 1) ? &maps.v : &maps.k, c0 + r, kvh, bar(kFull + j % R), lk - r, j & 1, failed, &g_packed_error);
      }
    }
  } else {
    more_regs<kComputeRegs>();
    const int t = warp >> 2, w = warp & 3, nt = t ? n1 : n0;
    const int row = row0 + t * kTile + w * 32 + lane, first = row0 + t * kTile + w * 32;
    const uint32_t ts = tmem + ((uint32_t)(32 * w) << 16) + kTile * t, to = ts + 256;
    // last key that this row sees, and that the warp's first row sees
    const int lim = min(a.causal ? row + off : lk - 1, lk - 1), lim_first = min(a.causal ? first + off : lk - 1, lk - 1);
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < nt; ++i) {
      wait_bar(bar(kSFull + t), i & 1, failed, &g_packed_error);
      fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int c = 0; c < kTile; c += 32) ld32(ts + c, x + c);
      wait_ld(x);
      const int kb = i * kTile;
      if (kb + kTile - 1 > lim_first) {
#pragma unroll
        for (int c = 0; c < kTile; ++c) if (kb + c > lim) x[c] = 0xff800000u;
      }
      float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
      for (int c = 0; c < kTile; c += 4) {
        m0 = fmaxf(m0, __uint_as_float(x[c])); m1 = fmaxf(m1, __uint_as_float(x[c + 1]));
        m2 = fmaxf(m2, __uint_as_float(x[c + 2])); m3 = fmaxf(m3, __uint_as_float(x[c + 3]));
      }
      const float mn = fmaxf(m, fmaxf(fmaxf(m0, m1), fmaxf(m2, m3)) * a.scale_log2);
      const bool raise = mn > m + 8.f;      // true where there was none yet
      if (__any_sync(0xffffffffu, raise)) {
        const float f = raise ? pow2(m - mn) : 1.f;
        if (raise) m = mn;
        l *= f;
        if (i > 0) {
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
      const float u = m == -INFINITY ? 0.f : -m;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y0 = pow2(fmaf(__uint_as_float(x[c + 2 * e]), a.scale_log2, u)), y1 = pow2(fmaf(__uint_as_float(x[c + 2 * e + 1]), a.scale_log2, u));
          l0 += y0; l1 += y1;
          p[e] = packed::Half<T>::pack(y0, y1);
        }
        st16(ts + c / 2, p);
      }
      l += l0 + l1;
      wait_st();
      fence_before();
      arrive(bar(kPFull + t));
    }
    if (nt > 0) {
      wait_bar(bar(kOFull + t), 0, failed, &g_packed_error);
      fence_after();
    }
    const bool there = row < lq, bad = *failed;
    const float inv = bad ? NAN : l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    T* dst = static_cast<T*>(a.out) + ((long long)(q0 + row) * a.hq + h) * d;
    for (int c = 0; c < d; c += 16) {
      uint32_t o[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = 0;
      if (nt > 0) { ld16(to + c, o); wait_ld(o); }
      uint32_t p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = packed::Half<T>::pack(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
      if (there) {
        *reinterpret_cast<uint4*>(dst + c) = make_uint4(p[0], p[1], p[2], p[3]);
        *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(p[4], p[5], p[6], p[7]);
      }
    }
    if (there && a.lse) a.lse[(long long)h * a.nq + q0 + row] = bad ? NAN : l == 0.f ? -INFINITY : m * kLn2 + logf(l);
    fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem); }
}

// ---- reverse: dq ----------------------------------------------------------------------------------------------------
// 128 queries of one head.  Tensor memory: logits at 0, dP at 128 (dS replaces it, in two halves), dq at 256.  The two groups of four warps
// have 64 columns each of every row.  The next tile's logits are made as soon as these have been read, so that its exponentials run
// beside the products dS k and g v^T.
enum DqBar { kdqFull, kdqEmpty = kdqFull + 8, kdqQ = kdqEmpty + 8, kdqS, kdqSRead, kdqDp, kdqDs, kdqOut, kdqFix, kDqBars };

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) dq_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d, subs = d > 64 ? 2 : 1, tile_bytes = subs * kSub, R = ring_slots(subs);
  Tail* tail = reinterpret_cast<Tail*>(smem + (2 + R) * tile_bytes);
  const uint32_t sq = smem_addr(smem), sg = sq + tile_bytes, ring = sg + tile_bytes, bar0 = smem_addr(tail->bars);
  volatile int* failed = &tail->failed;
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 item = a.items[blockIdx.x];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int h = blockIdx.y, kvh = h / a.group, row0 = item.y * kTile, off = lk - lq, n = (item.w + kTile - 1) / kTile;
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kDqBars; ++i) init_bar(bar(i), i == kdqSRead || i == kdqDs ? 256 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;

  if (warp >= kMmaWarp) {
    fewer_regs<kOtherRegs>();
    if (warp == kMmaWarp && n > 0) {
      const uint32_t on = elect_one();
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };
      auto ready = [&](int j) { wait_bar(bar(kdqFull + j % R), (j / R) & 1, failed, &g_packed_error); fence_after(); };
      auto give = [&](int j) { if (j + R < 2 * n) commit(on, bar(kdqEmpty + j % R)); };
      wait_bar(bar(kdqQ), 0, failed, &g_packed_error);
      ready(0);
      product_rows<T>(on, tmem, sq, slot(0), d);
      commit(on, bar(kdqS));
      ready(1);
      product_rows<T>(on, tmem + kTile, sg, slot(1), d);
      commit(on, bar(kdqDp));
      give(1);
      for (int i = 0; i < n; ++i) {
        if (i + 1 < n) {
          ready(2 * i + 2);
          wait_bar(bar(kdqSRead), i & 1, failed, &g_packed_error);
          fence_after();
          product_rows<T>(on, tmem, sq, slot(2 * i + 2), d);
          commit(on, bar(kdqS));
        }
        wait_bar(bar(kdqDs), i & 1, failed, &g_packed_error);
        fence_after();
        product_cols<T>(on, tmem + 256, tmem + kTile, 64, slot(2 * i), d, i > 0);
        give(2 * i);
        if (i + 1 < n) {
          ready(2 * i + 3);
          product_rows<T>(on, tmem + kTile, sg, slot(2 * i + 3), d);
          commit(on, bar(kdqDp));
          give(2 * i + 3);
        }
      }
      commit(on, bar(kdqOut));
    } else if (warp == kLoadWarp && n > 0) {
      Loader ld{lane, subs, bar(kdqFix)};
      if (lane == 0) {
        expect(bar(kdqQ), 2 * tile_bytes);
        ld.copies(sq, &maps.q, q0 + row0, h, bar(kdqQ));
        ld.copies(sg, &maps.g, q0 + row0, h, bar(kdqQ));
      }
      __syncwarp();
      for (int j = 0; j < 2 * n; ++j) {
        if (j >= R) wait_bar(bar(kdqEmpty + j % R), (j / R - 1) & 1, failed, &g_packed_error);
        const int r = (j >> 1) * kTile;
        ld.tile(ring + (j % R) * tile_bytes, (j & 1) ? &maps.v : &maps.k, c0 + r, kvh, bar(kdqFull + j % R), lk - r, !(j & 1), failed, &g_packed_error);
      }
    }
  } else {
    more_regs<kComputeRegs>();
    const int half = warp >> 2, w = warp & 3, row = row0 + w * 32 + lane, first = row0 + w * 32, col = 64 * half;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w) << 16);
    const int lim = min(a.causal ? row + off : lk - 1, lk - 1), lim_first = min(a.causal ? first + off : lk - 1, lk - 1);
    const long long at = (long long)h * a.nq + q0 + row;
    const bool there = row < lq;
    const float e = there ? -a.lse[at] * kLog2e : -INFINITY, delta = there ? a.delta[at] : 0.f;
    for (int i = 0; i < n; ++i) {
      uint32_t x[64], y[64];
      wait_bar(bar(kdqS), i & 1, failed, &g_packed_error);
      fence_after();
      ld32(lanes + col, x);
      ld32(lanes + col + 32, x + 32);
      wait_ld(x);
      fence_before();
      arrive(bar(kdqSRead));
#pragma unroll
      for (int c = 0; c < 64; ++c) x[c] = __float_as_uint(pow2(fmaf(__uint_as_float(x[c]), a.scale_log2, e)));
      const int kb = i * kTile + col;
      wait_bar(bar(kdqDp), i & 1, failed, &g_packed_error);
      fence_after();
      ld32(lanes + kTile + col, y);
      ld32(lanes + kTile + col + 32, y + 32);
      wait_ld(y);
#pragma unroll
      for (int c = 0; c < 64; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) * (__uint_as_float(y[c]) - delta));
      if (kb + 63 > lim_first) {
#pragma unroll
        for (int c = 0; c < 64; ++c) if (kb + c > lim) x[c] = 0;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) y[c] = packed::Half<T>::pack(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1]));
      st16(lanes + kTile + col, y);
      st16(lanes + kTile + col + 16, y + 16);
      wait_st();
      fence_before();
      arrive(bar(kdqDs));
    }
    if (n > 0) {
      wait_bar(bar(kdqOut), 0, failed, &g_packed_error);
      fence_after();
    }
    const float f = *failed ? NAN : a.scale;
    T* dst = static_cast<T*>(a.dq) + ((long long)(q0 + row) * a.hq + h) * d;
    for (int c = 16 * half; c < d; c += 32) {
      uint32_t o[16], p[8];
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k] = 0;
      if (n > 0) { ld16(lanes + 256 + c, o); wait_ld(o); }
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] = packed::Half<T>::pack(__uint_as_float(o[2 * k]) * f, __uint_as_float(o[2 * k + 1]) * f);
      if (there) {
        *reinterpret_cast<uint4*>(dst + c) = make_uint4(p[0], p[1], p[2], p[3]);
        *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(p[4], p[5], p[6], p[7]);
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem); }
}

// ---- reverse: dk and dv ---------------------------------------------------------------------------------------------
// 128 keys of one key head: rows of the products are keys, columns the queries of all heads of the group, 128 at a time.  Tensor memory:
// logits at 0 (P replaces them), dP at 128 (dS replaces it), dv at 256, dk at 384.  The tensor cores work in the order
// dv(i), logits(i + 1), dk(i), dP(i + 1): each pair runs beside the other half of the elementwise work.
enum DkvBar { kkvFull, kkvEmpty = kkvFull + 8, kkvK = kkvEmpty + 8, kkvS, kkvP, kkvDp, kkvDs, kkvOut, kkvFix, kkvStat, kkvStatFree = kkvStat + 2,
              kDkvBars = kkvStatFree + 2 };

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) dkv_kernel(const PackedArgs a, const __grid_constant__ Maps maps) {
  extern __shared__ unsigned char raw[];
  unsigned char* smem = aligned_smem(raw);
  const int d = a.d, subs = d > 64 ? 2 : 1, tile_bytes = subs * kSub, R = ring_slots(subs);
  float* stats = reinterpret_cast<float*>(smem + (2 + R) * tile_bytes);      // [2][128] -lse in log2, [2][128] -delta
  Tail* tail = reinterpret_cast<Tail*>(stats + 4 * kTile);
  const uint32_t sk = smem_addr(smem), sv = sk + tile_bytes, ring = sv + tile_bytes, bar0 = smem_addr(tail->bars);
  volatile int* failed = &tail->failed;
  auto bar = [&](int k) { return bar0 + 8 * k; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int4 item = a.items[blockIdx.x];
  const int s = item.x, q0 = a.start_q[s], lq = a.start_q[s + 1] - q0, c0 = a.start_kv[s], lk = a.start_kv[s + 1] - c0;
  const int kvh = blockIdx.y, row0 = item.y * kTile, off = lk - lq, i0 = item.z;
  const int per = (max(lq - i0, 0) + kTile - 1) / kTile, n = per * a.group;
  if (warp == kMmaWarp) alloc_tmem(&tail->tmem);
  if (tid == 0) {
    tail->failed = 0;
    for (int i = 0; i < kDkvBars; ++i)
      init_bar(bar(i), i == kkvP || i == kkvDs ? 256 : i == kkvStat || i == kkvStat + 1 ? 64 : i == kkvStatFree || i == kkvStatFree + 1 ? 8 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tail->tmem;

  if (warp >= kMmaWarp) {
    fewer_regs<kOtherRegs>();
    if (warp == kMmaWarp && n > 0) {
      const uint32_t on = elect_one(), dv = tmem + 256, dk = tmem + 256 + kTile;
      auto slot = [&](int j) { return ring + (j % R) * tile_bytes; };      // queries 0, 2, .., cotangents 1, 3, ..
      auto ready = [&](int j) { wait_bar(bar(kkvFull + j % R), (j / R) & 1, failed, &g_packed_error); fence_after(); };
      auto give = [&](int j) { if (j + R < 2 * n) commit(on, bar(kkvEmpty + j % R)); };
      wait_bar(bar(kkvK), 0, failed, &g_packed_error);
      ready(0);
      product_rows<T>(on, tmem, sk, slot(0), d);
      commit(on, bar(kkvS));
      ready(1);
      product_rows<T>(on, tmem + kTile, sv, slot(1), d);
      commit(on, bar(kkvDp));
      for (int i = 0; i < n; ++i) {
        wait_bar(bar(kkvP), i & 1, failed, &g_packed_error);
        fence_after();
        product_cols<T>(on, dv, tmem, 64, slot(2 * i + 1), d, i > 0);
        give(2 * i + 1);
        if (i + 1 < n) {
          ready(2 * i + 2);
          product_rows<T>(on, tmem, sk, slot(2 * i + 2), d);
          commit(on, bar(kkvS));
        }
        wait_bar(bar(kkvDs), i & 1, failed, &g_packed_error);
        fence_after();
        product_cols<T>(on, dk, tmem + kTile, 64, slot(2 * i), d, i > 0);
        give(2 * i);
        if (i + 1 < n) {
          ready(2 * i + 3);
          product_rows<T>(on, tmem + kTile, sv, slot(2 * i + 3), d);
          commit(on, bar(kkvDp));
        }
      }
      commit(on, bar(kkvOut));
    } else if (warp == kLoadWarp && n > 0) {
      Loader ld{lane, subs, bar(kkvFix)};
      if (lane == 0) {
        expect(bar(kkvK), 2 * tile_bytes);
        ld.copies(sk, &maps.k, c0 + row0, kvh, bar(kkvK));
        ld.copies(sv, &maps.v, c0 + row0, kvh, bar(kkvK));
      }
      __syncwarp();
      for (int j = 0; j < 2 * n; ++j) {
        if (j >= R) wait_bar(bar(kkvEmpty + j % R), (j / R - 1) & 1, failed, &g_packed_error);
        const int i = j >> 1, hq = kvh * a.group + i / per, b = i0 + (i % per) * kTile;
        ld.tile(ring + (j % R) * tile_bytes, (j & 1) ? &maps.g : &maps.q, q0 + b, hq, bar(kkvFull + j % R), lq - b, true, failed, &g_packed_error);
      }
    } else if (warp > kLoadWarp) {
      const int r0 = (warp - kLoadWarp - 1) * 32 + lane;
      for (int i = 0; i < n; ++i) {
        const int st = i & 1, hq = kvh * a.group + i / per, b = i0 + (i % per) * kTile;
        if (i >= 2) wait_bar(bar(kkvStatFree + st), ((i >> 1) - 1) & 1, failed, &g_packed_error);
        for (int r = r0; r < kTile; r += 64) {
          const bool ok = b + r < lq;
          const long long at = (long long)hq * a.nq + q0 + b + r;
          stats[st * kTile + r] = ok ? fmaf(-a.lse[at], kLog2e, packed::prob_shift<T>()) : -INFINITY;
          stats[(2 + st) * kTile + r] = ok ? -a.delta[at] * packed::prob_unscale<T>() : 0.f;
        }
        arrive(bar(kkvStat + st));
      }
    }
  } else {
    more_regs<kComputeRegs>();
    const int half = warp >> 2, w = warp & 3, row = row0 + w * 32 + lane, last = row0 + w * 32 + 31, col = 64 * half;
    const uint32_t lanes = tmem + ((uint32_t)(32 * w) << 16);
    // first query that sees this key, and that sees the warp's last key
    const int lim = a.causal ? row - off : 0, lim_last = a.causal ? last - off : 0;
    for (int i = 0; i < n; ++i) {
      const int st = i & 1, ib = i0 + (i % per) * kTile + col;
      uint32_t x[64], y[64];
      wait_bar(bar(kkvStat + st), (i >> 1) & 1, failed, &g_packed_error);
      wait_bar(bar(kkvS), i & 1, failed, &g_packed_error);
      fence_after();
      ld32(lanes + col, x);
      ld32(lanes + col + 32, x + 32);
      wait_ld(x);
      const float4* e = reinterpret_cast<const float4*>(stats + st * kTile + col);
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float4 v = e[c];
        x[4 * c] = __float_as_uint(pow2(fmaf(__uint_as_float(x[4 * c]), a.scale_log2, v.x)));
        x[4 * c + 1] = __float_as_uint(pow2(fmaf(__uint_as_float(x[4 * c + 1]), a.scale_log2, v.y)));
        x[4 * c + 2] = __float_as_uint(pow2(fmaf(__uint_as_float(x[4 * c + 2]), a.scale_log2, v.z)));
        x[4 * c + 3] = __float_as_uint(pow2(fmaf(__uint_as_float(x[4 * c + 3]), a.scale_log2, v.w)));
      }
      if (a.causal && ib < lim_last) {
#pragma unroll
        for (int c = 0; c < 64; ++c) if (ib + c < lim) x[c] = 0;
      }
#pragma unroll
      for (int c = 0; c < 32; ++c) y[c] = packed::Half<T>::pack(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1]));
      st16(lanes + col, y);
      st16(lanes + col + 16, y + 16);
      wait_st();
      fence_before();
      arrive(bar(kkvP));
      wait_bar(bar(kkvDp), i & 1, failed, &g_packed_error);
      fence_after();
      ld32(lanes + kTile + col, y);
      ld32(lanes + kTile + col + 32, y + 32);
      wait_ld(y);
      const float4* dl = reinterpret_cast<const float4*>(stats + (2 + st) * kTile + col);
      constexpr float un = packed::prob_unscale<T>();
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const float4 v = dl[c];
        const float s0 = __uint_as_float(x[4 * c]) * fmaf(__uint_as_float(y[4 * c]), un, v.x), s1 = __uint_as_float(x[4 * c + 1]) * fmaf(__uint_as_float(y[4 * c + 1]), un, v.y);
        const float s2 = __uint_as_float(x[4 * c + 2]) * fmaf(__uint_as_float(y[4 * c + 2]), un, v.z), s3 = __uint_as_float(x[4 * c + 3]) * fmaf(__uint_as_float(y[4 * c + 3]), un, v.w);
        y[2 * c] = packed::Half<T>::pack(s0, s1);
        y[2 * c + 1] = packed::Half<T>::pack(s2, s3);
      }
      __syncwarp();
      if (lane == 0) arrive(bar(kkvStatFree + st));
      st16(lanes + kTile + col, y);
      st16(lanes + kTile + col + 16, y + 16);
      wait_st();
      fence_before();
      arrive(bar(kkvDs));
    }
    if (n > 0) {
      wait_bar(bar(kkvOut), 0, failed, &g_packed_error);
      fence_after();
    }
    const bool there = row < lk, bad = *failed;
    const long long at = ((long long)(c0 + row) * a.hk + kvh) * d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float f = bad ? NAN : which ? a.scale : packed::prob_unscale<T>();
      T* dst = static_cast<T*>(which ? a.dk : a.dv) + at;
      for (int c = 16 * half; c < d; c += 32) {
        uint32_t o[16], p[8];
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = 0;
        if (n > 0) { ld16(lanes + 256 + which * kTile + c, o); wait_ld(o); }
#pragma unroll
        for (int k = 0; k < 8; ++k) p[k] = packed::Half<T>::pack(__uint_as_float(o[2 * k]) * f, __uint_as_float(o[2 * k + 1]) * f);
        if (there) {
          *reinterpret_cast<uint4*>(dst + c) = make_uint4(p[0], p[1], p[2], p[3]);
          *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(p[4], p[5], p[6], p[7]);
        }
      }
    }
    fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) { fence_after(); free_tmem(tmem); }
}

static_assert(kFwdBars <= 32 && kDqBars <= 32 && kDkvBars <= 32, "barriers");
int smem_bytes(int d, bool stats) { return 1024 + (d > 64 ? 6 * 2 : 10) * (int)kSub + (stats ? 4 * kTile * 4 : 0) + (int)sizeof(Tail); }

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
template <typename T> bool map_of(CUtensorMap* m, const Rows& r, long long rows, int heads, int d) {
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)heads};
  const cuuint64_t strides[2] = {(cuuint64_t)r.row * 2, (cuuint64_t)r.head * 2};
  const cuuint32_t box[3] = {64, kTile, 1}, ones[3] = {1, 1, 1};
  return encoder()(m, std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(r.p), dims,
                   strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <typename T> bool maps_of(Maps* m, const PackedArgs& a, bool reverse) {
  if (!encoder()) return false;
  return map_of<T>(&m->q, a.q, a.nq, a.hq, a.d) && map_of<T>(&m->k, a.k, a.nkv, a.hk, a.d) && map_of<T>(&m->v, a.v, a.nkv, a.hk, a.d) &&
         (reverse ? map_of<T>(&m->g, a.g, a.nq, a.hq, a.d) : (m->g = m->q, true));
}
template <typename K> int launch(K kernel, dim3 grid, bool stats, cudaStream_t st, const PackedArgs& a, const Maps& m) {
  const int smem = smem_bytes(a.d, stats);
  SO3LR_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kernel<<<grid, kThreads, smem, st>>>(a, m);
  count_launch();
  return kOk;
}

}  // namespace

template <typename T> int packed_forward_tc(cudaStream_t st, const PackedArgs& a, int n_items) {
  Maps m;
  if (!maps_of<T>(&m, a, false)) return kInvalidArgument;
  return launch(forward_kernel<T>, dim3(n_items, a.hq), false, st, a, m);
}
template <typename T> int packed_reverse_tc(cudaStream_t st, PackedArgs a, const int4* items_q, int n_q, const int4* items_kv, int n_kv) {
  Maps m;
  if (!maps_of<T>(&m, a, true)) return kInvalidArgument;
  a.items = items_q;
  const int rc = launch(dq_kernel<T>, dim3(n_q, a.hq), false, st, a, m);
  if (rc) return rc;
  a.items = items_kv;
  return launch(dkv_kernel<T>, dim3(n_kv, a.hk), true, st, a, m);
}
int packed_error(int* out) {
  const cudaError_t e = cudaMemcpyFromSymbol(out, g_packed_error, sizeof(int));
  return e == cudaSuccess ? kOk : kCudaError;
}

template int packed_forward_tc<__nv_bfloat16>(cudaStream_t, const PackedArgs&, int);
template int packed_forward_tc<__half>(cudaStream_t, const PackedArgs&, int);
template int packed_reverse_tc<__nv_bfloat16>(cudaStream_t, PackedArgs, const int4*, int, const int4*, int);
template int packed_reverse_tc<__half>(cudaStream_t, PackedArgs, const int4*, int, const int4*, int);

}  // namespace so3lr
