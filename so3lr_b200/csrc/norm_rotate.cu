// Queries and keys normalised per head and rotated by angles that are linear in the row's position, in one pass, and its reverse.
//
//   y = w x / sqrt(mean(x^2) + eps)  (without a norm: y = x),  theta_p = sum_a pos_a f_ap,
//   (o1, o2)_p = (y1 cos - y2 sin, y1 sin + y2 cos)_p          pairs (p, p + d/2) or (2p, 2p + 1)
// The product of two rotated rows depends on the difference of their positions only.  With one axis and f_p falling geometrically these are
// the usual positions of a sequence; with three axes they are the coordinates of an atom, and the gradient of the positions (a force) is
//   dtheta_p = sum over heads of (g2 o1 - g1 o2)_p,  dpos_a = sum_p f_ap dtheta_p.
// With gy = g rotated by -theta and xhat = x / sqrt(..):  dw = sum of gy xhat,  dx = (w gy - xhat mean(w gy xhat)) / sqrt(..).
//
// Bound by memory: forward reads and writes every value once, the reverse pass reads x and g and writes dx.  A thread owns 16 bytes of both
// halves of the pairs of one row (8 pairs of a 16-bit type, 4 of float32), so a row of 128 16-bit values takes 8 lanes, and walks over heads of
// one token; with few tokens the heads are spread over more threads (`slots`).  The cosines and sines of a CTA's tokens are formed
// once, spread over its threads, into shared memory: the angle is formed and reduced in double (the position of a far token times a
// frequency near one loses its fraction in float32), which costs more than all the rest of a row.
#include "../../include/so3lr_b200.h"

#include "kernels.h"
#include "packed_mma.cuh"

namespace so3lr {

struct RotateArgs {
  Rows x[2], g[2];                 // queries, keys; cotangents of the rotated rows
  void *out[2] = {}, *dx[2] = {};  // contiguous (n, heads, d)
  const void* w[2] = {};           // (d) weights of the norm, float32 or the rows' type
  void* dw[2] = {};
  const void* pos = nullptr;       // (n, axes) contiguous, float32 or float64
  const float* freq = nullptr;     // (axes, d / 2)
  void* dpos = nullptr;
  float* part = nullptr;           // (CTAs, 2, d) shares of dw
  int heads[2] = {}, n = 0, d = 0, axes = 0, norm = 0, w_f32 = 0, pos_f64 = 0, slots = 1;
  float eps = 0.f;
};

namespace {

constexpr int kThreads = 256;

// 16 bytes of T as floats and back
template <typename T> struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  static __device__ __forceinline__ void load(uint4 u, float* f) {
    const uint32_t s[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) { const float2 v = packed::Half<T>::unpack(s[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
      else f[i] = __uint_as_float(s[i]);
    }
  }
  static __device__ __forceinline__ uint4 store(const float* f) {
    uint32_t s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) s[i] = packed::Half<T>::pack(f[2 * i], f[2 * i + 1]);
      else s[i] = __float_as_uint(f[i]);
    }
    return make_uint4(s[0], s[1], s[2], s[3]);
  }
};

// A thread's values of a row: two 16-byte pieces at offsets off_a, off_b; a[i] and b[i] form pair p0 + i.
template <typename T, bool NEIGHBORS> struct Piece {
  static constexpr int N = Vec<T>::N;
  static __device__ __forceinline__ int off_a(int part, int d) { return NEIGHBORS ? part * 2 * N : part * N; }
  static __device__ __forceinline__ int off_b(int part, int d) { return NEIGHBORS ? part * 2 * N + N : part * N + d / 2; }
  static __device__ __forceinline__ void split(uint4 u, uint4 v, float* a, float* b) {
    if constexpr (NEIGHBORS) {
      float f[2 * N];
      Vec<T>::load(u, f); Vec<T>::load(v, f + N);
#pragma unroll
      for (int i = 0; i < N; ++i) { a[i] = f[2 * i]; b[i] = f[2 * i + 1]; }
    } else {
      Vec<T>::load(u, a); Vec<T>::load(v, b);
    }
  }
  static __device__ __forceinline__ void join(const float* a, const float* b, uint4& u, uint4& v) {
    if constexpr (NEIGHBORS) {
      float f[2 * N];
#pragma unroll
      for (int i = 0; i < N; ++i) { f[2 * i] = a[i]; f[2 * i + 1] = b[i]; }
      u = Vec<T>::store(f); v = Vec<T>::store(f + N);
    } else {
      u = Vec<T>::store(a); v = Vec<T>::store(b);
    }
  }
};

// cos and sin of theta: reduced to x in [-pi/4, pi/4] in double, so that one rounding to float32 costs 2^-25 of an angle below one, then
// x + x^3 P(x^2) and 1 - x^2/2 + x^4 Q(x^2) with P and Q of degree 2 fitted for the least largest error there (1.8e-9 and 1e-10; least
// squares reweighted by the error).  The library's pair carries its reduction of large arguments along (32,771 rows of 40 heads x
// 128: 139 us with it, 131 without).  Beyond 2^53 nothing is left of an angle: where the reduction fails there, the row stays unturned.
__device__ __forceinline__ void cos_sin(double theta, float& c, float& s) {
  const double n = rint(theta * 0.6366197723675814);
  const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, theta));
  const int q = (int)((long long)n & 3);
  float x = (float)r;
  if (fabsf(x) > 1.f) x *= 0.f;      // infinite ones become NaN
  const float z = x * x;
  const float sr = fmaf(x * z, fmaf(z, fmaf(z, -1.9495567539706826e-4f, 8.331977762281895e-3f), -0.16666650772094727f), x);
  const float cr = fmaf(z * z, fmaf(z, fmaf(z, 2.4438379114144482e-5f, -1.3887366512790322e-3f), 4.166664555668831e-2f), fmaf(z, -0.5f, 1.f));
  c = (q & 1) ? sr : cr; s = (q & 1) ? cr : sr;
  if (q == 1 || q == 2) c = -c;
  if (q >= 2) s = -s;
}

// cosines and sines of `tokens` tokens from t0 on, (tokens, d / 2), by the whole CTA
__device__ __forceinline__ void angle_table(const RotateArgs& A, int t0, int tokens, float* c, float* s) {
  const int half = A.d / 2;
  for (int e = threadIdx.x; e < tokens * half; e += kThreads) {
    const int token = t0 + e / half, p = e % half;
    float cc = 1.f, ss = 0.f;
    if (token < A.n && A.axes) {
      double th = 0.0;
      for (int a = 0; a < A.axes; ++a) {
        const size_t at = (size_t)token * A.axes + a;
        const double x = A.pos_f64 ? static_cast<const double*>(A.pos)[at] : (double)static_cast<const float*>(A.pos)[at];
        th = fma(x, (double)A.freq[(size_t)a * half + p], th);
      }
      cos_sin(th, cc, ss);
    }
    c[e] = cc; s[e] = ss;
  }
}
// N floats of shared memory
template <int N>
__device__ __forceinline__ void take(const float* table, int at, float* out) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(table + at + i);
    out[i] = v.x; out[i + 1] = v.y; out[i + 2] = v.z; out[i + 3] = v.w;
  }
}

// weights of both sides (2, d) into shared memory, in the order of the threads' pieces: those of a piece's a values, then of its b values
template <typename T, bool NEIGHBORS>
__device__ __forceinline__ void weight_table(const RotateArgs& A, float* w) {
  constexpr int N = Vec<T>::N;
  for (int e = threadIdx.x; e < 2 * A.d; e += kThreads) {
    const int side = e / A.d, i = e % A.d, part = i / (2 * N), k = i % (2 * N), p = part * N + k % N, second = k / N;
    const int at = NEIGHBORS ? 2 * p + second : p + second * (A.d / 2);
    if (A.w[side]) w[e] = A.w_f32 ? static_cast<const float*>(A.w[side])[at] : (float)static_cast<const T*>(A.w[side])[at];
  }
}

// Heads of queries and keys as one range [0, heads of both): side, row piece and weights of head h
template <typename T> struct Head {
  int side, h;
  bool there;
  __device__ __forceinline__ Head(const RotateArgs& A, int i) : side(i >= A.heads[0]), h(i - (i >= A.heads[0] ? A.heads[0] : 0)), there(i < A.heads[0] + A.heads[1]) {}
};

// W lanes per row (the next power of two of the parts), `slots` heads of a token side by side, then tokens.  The next heads' rows are
// asked for before the present ones are worked on, the first ones before the angles are formed.
template <typename T, bool NEIGHBORS, bool NORM, int U>
__global__ void __launch_bounds__(kThreads, 4) forward_kernel(const RotateArgs A, int W) {
  using P = Piece<T, NEIGHBORS>;
  constexpr int N = Vec<T>::N;
  const int part = threadIdx.x % W, group = threadIdx.x / W, slot = group % A.slots;
  const int per = kThreads / W / A.slots, token = blockIdx.x * per + group / A.slots, heads = A.heads[0] + A.heads[1];
  const bool on = token < A.n && part * N < A.d / 2;
  const int oa = P::off_a(part, A.d), ob = P::off_b(part, A.d);
  extern __shared__ __align__(16) float table[];
  uint4 u[U], v[U];
  auto load = [&](int hb) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Head<T> h(A, hb + slot + k * A.slots);
      u[k] = v[k] = make_uint4(0, 0, 0, 0);
      if (on && h.there) {
        const T* src = static_cast<const T*>(A.x[h.side].p) + (long long)token * A.x[h.side].row + h.h * A.x[h.side].head;
        u[k] = __ldcs(reinterpret_cast<const uint4*>(src + oa));
        v[k] = __ldcs(reinterpret_cast<const uint4*>(src + ob));
      }
    }
  };
  load(0);
  float c[N], s[N];
  if (NORM) weight_table<T, NEIGHBORS>(A, table + per * A.d);
  angle_table(A, blockIdx.x * per, per, table, table + per * (A.d / 2));
  __syncthreads();
  if (on) {
    const int at = (group / A.slots) * (A.d / 2) + part * N;
    take<N>(table, at, c);
    take<N>(table + per * (A.d / 2), at, s);
  }
  for (int hb = 0; hb < heads; hb += U * A.slots) {      // the same trips for all lanes: the sums below are over a warp
    float a[U][N], b[U][N];
#pragma unroll
    for (int k = 0; k < U; ++k) P::split(u[k], v[k], a[k], b[k]);
    if (hb + U * A.slots < heads) load(hb + U * A.slots);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const Head<T> h(A, hb + slot + k * A.slots);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(a[k][i], a[k][i], fmaf(b[k][i], b[k][i], ss));
        for (int o = W >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = 1.f / sqrtf(ss / A.d + A.eps);
        if (on) {
          const float* w = table + per * A.d + h.side * A.d + part * 2 * N;
          float wa[N], wb[N];
          take<N>(w, 0, wa);
          take<N>(w, N, wb);
#pragma unroll
          for (int i = 0; i < N; ++i) { a[k][i] *= r * wa[i]; b[k][i] *= r * wb[i]; }
        }
      }
      if (on && h.there) {
        T* dst = static_cast<T*>(A.out[h.side]) + ((long long)token * A.heads[h.side] + h.h) * A.d;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float t = a[k][i] * c[i] - b[k][i] * s[i];
          b[k][i] = a[k][i] * s[i] + b[k][i] * c[i];
          a[k][i] = t;
        }
        uint4 x, y;
        P::join(a[k], b[k], x, y);
        *reinterpret_cast<uint4*>(dst + oa) = x;
        *reinterpret_cast<uint4*>(dst + ob) = y;
      }
    }
  }
}

// CTAs walk over tiles of tokens; the shares of dw of a CTA end in one row of A.part.  The sums have a fixed order.
template <typename T, bool NEIGHBORS, bool NORM>
__global__ void __launch_bounds__(kThreads, 3) reverse_kernel(const RotateArgs A, int W) {
  using P = Piece<T, NEIGHBORS>;
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(16) float table[];
  __shared__ float th[kThreads * N];                     // dtheta of every thread
  __shared__ float sw[kThreads / 32][2 * N * 32];        // dw of the warps, one side at a time
  const int part = threadIdx.x % W, group = threadIdx.x / W, slot = group % A.slots, per = kThreads / W / A.slots, heads = A.heads[0] + A.heads[1];
  const bool there = part * N < A.d / 2;
  const int oa = P::off_a(part, A.d), ob = P::off_b(part, A.d);
  float dwa[2][N], dwb[2][N];
#pragma unroll
  for (int i = 0; i < N; ++i) dwa[0][i] = dwa[1][i] = dwb[0][i] = dwb[1][i] = 0.f;
  if (NORM) weight_table<T, NEIGHBORS>(A, table + per * A.d);
  uint4 u, v, gu, gv;
  auto load = [&](int token, int hb) {
    const Head<T> h(A, hb + slot);
    u = v = gu = gv = make_uint4(0, 0, 0, 0);
    if (token < A.n && there && h.there) {
      const T* src = static_cast<const T*>(A.x[h.side].p) + (long long)token * A.x[h.side].row + h.h * A.x[h.side].head;
      const T* gsrc = static_cast<const T*>(A.g[h.side].p) + (long long)token * A.g[h.side].row + h.h * A.g[h.side].head;
      u = __ldcs(reinterpret_cast<const uint4*>(src + oa));
      v = __ldcs(reinterpret_cast<const uint4*>(src + ob));
      gu = __ldcs(reinterpret_cast<const uint4*>(gsrc + oa));
      gv = __ldcs(reinterpret_cast<const uint4*>(gsrc + ob));
    }
  };
  for (int t0 = blockIdx.x * per; t0 < A.n; t0 += gridDim.x * per) {
    const int token = t0 + group / A.slots;
    const bool on = token < A.n && there;
    load(token, 0);
    float c[N], s[N], dth[N];
#pragma unroll
    for (int i = 0; i < N; ++i) dth[i] = 0.f;
    angle_table(A, t0, per, table, table + per * (A.d / 2));
    __syncthreads();
    if (on) {
      const int at = (group / A.slots) * (A.d / 2) + part * N;
      take<N>(table, at, c);
      take<N>(table + per * (A.d / 2), at, s);
    }
    for (int hb = 0; hb < heads; hb += A.slots) {      // the same trips for all lanes: the sums below are over a warp
      const Head<T> h(A, hb + slot);
      float a[N], b[N], ga[N], gb[N];
      P::split(u, v, a, b);
      P::split(gu, gv, ga, gb);
      if (hb + A.slots < heads) load(token, hb + A.slots);
      float r = 1.f, dot = 0.f;
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
        for (int o = W >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = 1.f / sqrtf(ss / A.d + A.eps);
      }
      if (on && h.there) {      // a head that is not there has neither weights nor, with eps = 0, a finite norm
        float wa[N], wb[N];
        if (NORM) {
          const float* w = table + per * A.d + h.side * A.d + part * 2 * N;
          take<N>(w, 0, wa);
          take<N>(w, N, wb);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xa = a[i] * r, xb = b[i] * r, ya = NORM ? xa * wa[i] : xa, yb = NORM ? xb * wb[i] : xb;
          const float o1 = ya * c[i] - yb * s[i], o2 = ya * s[i] + yb * c[i];
          dth[i] = fmaf(gb[i], o1, fmaf(-ga[i], o2, dth[i]));
          float va = ga[i] * c[i] + gb[i] * s[i], vb = gb[i] * c[i] - ga[i] * s[i];
          if (NORM) {
            const float pa = va * xa, pb = vb * xb;
            if (h.side) { dwa[1][i] += pa; dwb[1][i] += pb; } else { dwa[0][i] += pa; dwb[0][i] += pb; }
            va *= wa[i]; vb *= wb[i];
            dot = fmaf(va, xa, fmaf(vb, xb, dot));
          }
          a[i] = xa; b[i] = xb; ga[i] = va; gb[i] = vb;
        }
      }
      if (NORM) {
        for (int o = W >> 1; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        dot /= A.d;
      }
      if (on && h.there) {
        T* dst = static_cast<T*>(A.dx[h.side]) + ((long long)token * A.heads[h.side] + h.h) * A.d;
        if (NORM) {
#pragma unroll
          for (int i = 0; i < N; ++i) { ga[i] = r * (ga[i] - a[i] * dot); gb[i] = r * (gb[i] - b[i] * dot); }
        }
        uint4 x, y;
        P::join(ga, gb, x, y);
        *reinterpret_cast<uint4*>(dst + oa) = x;
        *reinterpret_cast<uint4*>(dst + ob) = y;
      }
    }
    if (A.dpos) {
      // shares of the slots meet in shared memory; the first slot's lanes sum them, times the frequencies
#pragma unroll
      for (int i = 0; i < N; ++i) th[i * kThreads + threadIdx.x] = on ? dth[i] : 0.f;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dth[i] = 0.f;
        if (slot == 0) for (int k = 0; k < A.slots; ++k) dth[i] += th[i * kThreads + threadIdx.x + k * W];
      }
      for (int a = 0; a < A.axes; ++a) {
        float sum = 0.f;
        if (on && slot == 0) {
          const float* f = A.freq + (size_t)a * (A.d / 2) + part * N;
#pragma unroll
          for (int i = 0; i < N; ++i) sum = fmaf(f[i], dth[i], sum);
        }
        for (int o = W >> 1; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (token < A.n && slot == 0 && part == 0) {
          const size_t at = (size_t)token * A.axes + a;
          if (A.pos_f64) static_cast<double*>(A.dpos)[at] = sum; else static_cast<float*>(A.dpos)[at] = sum;
        }
      }
    }
    __syncthreads();      // the tables are written again
  }
  if constexpr (NORM) {
    if (!A.part) return;
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      // lanes with the same part of the row
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x = there ? dwa[side][i] : 0.f, y = there ? dwb[side][i] : 0.f;
        for (int o = W; o < 32; o <<= 1) { x += __shfl_xor_sync(0xffffffffu, x, o); y += __shfl_xor_sync(0xffffffffu, y, o); }
        const int lane = threadIdx.x & 31;
        if (lane < W) { sw[threadIdx.x >> 5][(2 * i) * 32 + lane] = x; sw[threadIdx.x >> 5][(2 * i + 1) * 32 + lane] = y; }
      }
      __syncthreads();
      for (int e = threadIdx.x; e < 2 * N * W; e += kThreads) {
        const int pt = e % W, i = (e / W) >> 1, second = (e / W) & 1, p = pt * N + i;
        if (p < A.d / 2) {
          float sum = 0.f;
          for (int w = 0; w < kThreads / 32; ++w) sum += sw[w][(2 * i + second) * 32 + pt];
          const int at = NEIGHBORS ? 2 * p + second : p + second * (A.d / 2);
          A.part[((size_t)blockIdx.x * 2 + side) * A.d + at] = sum;
        }
      }
      __syncthreads();
    }
  }
}

// dw: 32 columns per CTA, eight threads each over the CTAs' shares
template <typename T>
__global__ void __launch_bounds__(256) weight_kernel(const RotateArgs A, int rows) {
  __shared__ float sum[8][32];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
  float s = 0.f;
  if (col < 2 * A.d) for (int r = k; r < rows; r += 8) s += A.part[(size_t)r * 2 * A.d + col];
  sum[k][threadIdx.x & 31] = s;
  __syncthreads();
  if (k == 0 && col < 2 * A.d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += sum[i][threadIdx.x];
    const int side = col / A.d, i = col % A.d;
    if (A.dw[side]) {
      if (A.w_f32) static_cast<float*>(A.dw[side])[i] = s; else static_cast<T*>(A.dw[side])[i] = (T)s;
    }
  }
}

int next_pow2(int x) { int p = 1; while (p < x) p <<= 1; return p; }
// Lanes per row, and heads of a token that run side by side: as few as give every SM `busy` threads.  A thread with several heads asks for
// the next one's rows while it works on the present one, and the angles of a token are formed once for all of them; more threads hide more.
// 32,771 rows of 40 heads x 128 forward, busy 2,048 / 4,096 / 8,192: 140 / 131 / 140 us (5.1 TB/s; a copy of the bytes takes 103; with more than
// four CTAs on an SM the registers spill: 198); 16,411 rows of 32 heads x 64 reverse, 512 / 1,024 / 2,048: 56 / 47 / 53 us; 12,803 rows
// of 8 heads x 32 float32 reverse: 16 / 19 / 28.
void shape(RotateArgs& A, int value_bytes, bool reverse, int& W) {
  W = next_pow2(A.d / 2 / (16 / value_bytes));
  const int heads = A.heads[0] + A.heads[1];
  const int most = next_pow2(heads < 1 ? 1 : heads) < kThreads / W ? next_pow2(heads < 1 ? 1 : heads) : kThreads / W;
  const long long busy = reverse ? 1024 : 4096;
  A.slots = 1;
  while (A.slots < most && (long long)A.n * W * A.slots < busy * sm_count()) A.slots <<= 1;
}

template <typename T, bool NEIGHBORS, bool NORM>
void rotate_launch(cudaStream_t st, RotateArgs A, bool reverse, int grid_max) {
  int W;
  shape(A, sizeof(T), reverse, W);
  const int per = kThreads / W / A.slots, tiles = (A.n + per - 1) / per, smem = (per + 2) * A.d * (int)sizeof(float);
  if (!reverse) {
    forward_kernel<T, NEIGHBORS, NORM, 1><<<tiles, kThreads, smem, st>>>(A, W);
    count_launch();
    return;
  }
  const int grid = tiles < grid_max ? tiles : grid_max;
  reverse_kernel<T, NEIGHBORS, NORM><<<grid, kThreads, smem, st>>>(A, W);
  count_launch();
  if (A.part) {
    weight_kernel<T><<<(2 * A.d + 31) / 32, 256, 0, st>>>(A, grid);
    count_launch();
  }
}

template <typename T>
void rotate_typed(cudaStream_t st, const RotateArgs& A, bool neighbors, bool reverse, int grid_max) {
  if (neighbors) {
    if (A.norm) rotate_launch<T, true, true>(st, A, reverse, grid_max); else rotate_launch<T, true, false>(st, A, reverse, grid_max);
  } else {
    if (A.norm) rotate_launch<T, false, true>(st, A, reverse, grid_max); else rotate_launch<T, false, false>(st, A, reverse, grid_max);
  }
}
void rotate(cudaStream_t st, const RotateArgs& A, int type, bool neighbors, bool reverse, int grid_max) {
  if (type == kBF16) rotate_typed<__nv_bfloat16>(st, A, neighbors, reverse, grid_max);
  else if (type == kF16) rotate_typed<__half>(st, A, neighbors, reverse, grid_max);
  else rotate_typed<float>(st, A, neighbors, reverse, grid_max);
}

bool rows_ok(const so3lr_b200_rows* r, int type, int heads) {
  if (heads == 0) return true;
  const long long unit = type == kF32 ? 4 : 8;
  return r && r->data && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride % unit == 0 && r->head_stride % unit == 0;
}
Rows rows_of(const so3lr_b200_rows* r) { return r ? Rows{r->data, r->row_stride, r->head_stride} : Rows{}; }
int grid_limit() { return 3 * sm_count(); }      // CTAs of the reverse kernel that are resident at a time

}  // namespace
}  // namespace so3lr

using namespace so3lr;

extern "C" {

int so3lr_b200_norm_rotate(void* stream, const so3lr_b200_norm_rotate_args* a, const so3lr_b200_rows* q, const so3lr_b200_rows* k,
                           void* out_q, void* out_k) {
  if (!a || a->n < 0 || a->n > 0x7ff00000 || a->type < 0 || a->type > 2 || a->d < 16 || a->d > 256 || a->d % 16 || a->heads_q < 0 || a->heads_k < 0 || a->axes < 0 ||
      a->axes > 16 || (a->axes && a->n && (!a->positions || !a->frequencies)))
    return kInvalidArgument;
  if (a->n == 0 || a->heads_q + a->heads_k == 0) return kOk;
  if (!rows_ok(q, a->type, a->heads_q) || !rows_ok(k, a->type, a->heads_k) || (a->heads_q && !out_q) || (a->heads_k && !out_k)) return kInvalidArgument;
  if (a->norm && ((a->heads_q && !a->weight_q) || (a->heads_k && !a->weight_k))) return kInvalidArgument;
  RotateArgs A;
  A.x[0] = rows_of(q); A.x[1] = rows_of(k);
  A.out[0] = out_q; A.out[1] = out_k; A.w[0] = a->weight_q; A.w[1] = a->weight_k;
  A.pos = a->positions; A.freq = a->frequencies; A.heads[0] = a->heads_q; A.heads[1] = a->heads_k;
  A.n = a->n; A.d = a->d; A.axes = a->axes; A.norm = a->norm; A.w_f32 = a->weights_f32; A.pos_f64 = a->positions_f64; A.eps = a->eps;
  rotate(static_cast<cudaStream_t>(stream), A, a->type, a->neighbors != 0, false, 0);
  SO3LR_CUDA_CHECK(cudaGetLastError());
  return kOk;
}

int64_t so3lr_b200_norm_rotate_workspace(int d) { return (int64_t)grid_limit() * 2 * d * (int64_t)sizeof(float); }

int so3lr_b200_norm_rotate_vjp(void* stream, const so3lr_b200_norm_rotate_args* a, const so3lr_b200_rows* q, const so3lr_b200_rows* k,
                               const so3lr_b200_rows* g_q, const so3lr_b200_rows* g_k, void* d_q, void* d_k, void* d_positions,
                               void* d_weight_q, void* d_weight_k, void* workspace, int64_t workspace_bytes) {
  if (!a || a->n < 0 || a->n > 0x7ff00000 || a->type < 0 || a->type > 2 || a->d < 16 || a->d > 256 || a->d % 16 || a->heads_q < 0 || a->heads_k < 0 || a->axes < 0 ||
      a->axes > 16 || (a->axes && a->n && (!a->positions || !a->frequencies)) || (d_positions && !a->axes))
    return kInvalidArgument;
  const bool want_w = a->norm && (d_weight_q || d_weight_k);
  if (want_w && (!workspace || workspace_bytes < so3lr_b200_norm_rotate_workspace(a->d))) return kInvalidArgument;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->n > 0 && a->heads_q + a->heads_k > 0) {
    if (!rows_ok(q, a->type, a->heads_q) || !rows_ok(k, a->type, a->heads_k) || !rows_ok(g_q, a->type, a->heads_q) ||
        !rows_ok(g_k, a->type, a->heads_k) || (a->heads_q && !d_q) || (a->heads_k && !d_k))
      return kInvalidArgument;
    if (a->norm && ((a->heads_q && !a->weight_q) || (a->heads_k && !a->weight_k))) return kInvalidArgument;
    RotateArgs A;
    A.x[0] = rows_of(q); A.x[1] = rows_of(k); A.g[0] = rows_of(g_q); A.g[1] = rows_of(g_k);
    A.dx[0] = d_q; A.dx[1] = d_k; A.w[0] = a->weight_q; A.w[1] = a->weight_k; A.dw[0] = d_weight_q; A.dw[1] = d_weight_k;
    A.pos = a->positions; A.freq = a->frequencies; A.dpos = d_positions; A.part = want_w ? static_cast<float*>(workspace) : nullptr;
    A.heads[0] = a->heads_q; A.heads[1] = a->heads_k;
    A.n = a->n; A.d = a->d; A.axes = a->axes; A.norm = a->norm; A.w_f32 = a->weights_f32; A.pos_f64 = a->positions_f64; A.eps = a->eps;
    rotate(st, A, a->type, a->neighbors != 0, true, grid_limit());
  } else {
    const size_t wb = (size_t)a->d * (a->weights_f32 || a->type == kF32 ? 4 : 2);
    if (want_w && d_weight_q) SO3LR_CUDA_CHECK(cudaMemsetAsync(d_weight_q, 0, wb, st));
    if (want_w && d_weight_k) SO3LR_CUDA_CHECK(cudaMemsetAsync(d_weight_k, 0, wb, st));
    if (d_positions && a->n) SO3LR_CUDA_CHECK(cudaMemsetAsync(d_positions, 0, (size_t)a->n * a->axes * (a->positions_f64 ? 8 : 4), st));
  }
  SO3LR_CUDA_CHECK(cudaGetLastError());
  return kOk;
}

}  // extern "C"
