// Attention inside the structures of a packed batch: arguments shared by its kernels (packed_mma.cuh, packed_tc.cu) and its host side
// (packed_attention.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "common.cuh"

namespace so3lr {

enum ValueType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

// Rows of a strided operand: element (row, head, 0) lies at p + row * row_stride + head * head_stride (in elements), its d values
// contiguous; p and both strides are multiples of 16 bytes.
struct Rows {
  const void* p = nullptr;
  long long row = 0, head = 0;
};

struct PackedArgs {
  Rows q, k, v, g, o;           // g: cotangent of the output; o: the output (reverse pass)
  void* out = nullptr;          // (nq, hq, d) contiguous
  void* out_rest = nullptr;     // (nq, hq, d) what rounding o to 16 bits left, or null
  float* lse = nullptr;         // (hq, nq) logarithm to base 2 of the sum of exponentials; -inf for a row without keys
  float* delta = nullptr;       // (hq, nq) sum over d of g * o
  void *dq = nullptr, *dk = nullptr, *dv = nullptr;   // contiguous
  const int *start_q = nullptr, *start_kv = nullptr;
  // one work item per CTA, head and piece: {structure, tile, first, last}; [first, last) are the rows of the other side that the tile meets
  const int4* items = nullptr;
  const int* split_first = nullptr;                   // items of structure s: [split_first[s], split_first[s + 1])
  float* part_o = nullptr;      // (item, hk, part_rows, DP) of the split form
  float2* part_ml = nullptr;    // (item, hk, part_rows): running maximum (in units of log2) and sum
  int part_rows = 0;            // most rows of a structure: tokens times heads of a group
  int pieces = 1;               // into which an item's walk is cut; each leaves its share in part_o (pieces, hq, nq, d) and part_ml, or
  float* share[3] = {};         // (reverse) in share: (pieces, rows, heads, d) of dq, dk, dv
  // reverse pass of float16 on the tensor cores, else null: bits of the largest |g| and of sqrt(d) times the largest |v_jc| (structure, key head, 2),
  // and |g| of every row (hq, nq)
  unsigned* largest = nullptr;
  float* size_g = nullptr;
  int structures = 0;
  int jobs = 0;                 // of the tensor-core kernels: items times heads times pieces
  int* error = nullptr;         // of the tensor-core kernels: host memory that tells of a wait that has run out, and how often one is tried
  int wait_tries = 0;
  int* queue = nullptr;         // jobs that were handed out besides each CTA's first (forward; dq, and dk and dv)
  int rows = 0, rows_kv = 0;    // of the layout
  int longest_kv = 0;           // keys of its longest structure
  int stages = 2, rev_stages = 2;         // buffers for the walked side in the warp-level kernels: one where all of it fits into it
  int tile_rows = 64;           // rows of a CTA there: 64 or 16
  int nq = 0, nkv = 0, hq = 0, hk = 0, group = 1, d = 0, causal = 0;
  float scale = 0.f, scale_log2 = 0.f;                // scale * log2(e): the softmax runs on powers of two
};

constexpr int kPackTile = 64;   // rows of a tile of the mma kernels

// float16 keeps its 11 bits between 2^-14 and 2^16 only, and dS = P (dP - delta) is as small as the cotangents of a mean loss over thousands
// of keys, or as large as those of a scaled one.  It goes into its products times a power of two, which leaves with the factor `scale` at their
// end: exact.  The warp-level kernels, whose sums are in registers, take it from the values (shift_rows).  On the tensor cores it is known ahead and
// costs no instruction: |dS| <= |g| |v| + |g| |o| <= 2 |g| sqrt(d) max |v_jc|, and the exponent that puts this bound into [2^14, 2^15) is a query
// row's own ahead of dS k, and one of a structure and key head ahead of dS^T q, which sums over queries.
template <typename T> constexpr bool kShifted = std::is_same<T, __half>::value;
// The forward kernels' probabilities relative to a row's largest take a power of two as well, so that what many keys far below the largest add up to
// is not lost in the last steps of float16: its largest number, 65504, leaves room for 2^15.  On the tensor cores the reference may lag behind
// the largest by a factor 2^kLag, for which room has to be left too.
template <typename T> constexpr float kLag = kShifted<T> ? 4.f : 8.f;
template <typename T, bool LAGS> constexpr float kHead = !kShifted<T> ? 0.f : LAGS ? 15.f - kLag<T> : 15.f;
__device__ __forceinline__ int grad_shift(float g, float v) {
  const float x = 2.f * g * v;
  return x > 0.f ? 14 - ((int)(__float_as_uint(x) >> 23) - 127) : 0;
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// kernels on the warp-level matrix instructions, one translation unit per type
template <typename T> int packed_forward_mma(cudaStream_t st, const PackedArgs& a, int n_items);
template <typename T> int packed_forward_split(cudaStream_t st, const PackedArgs& a, int n_items, int n_structures, bool combine);
template <typename T> int packed_dq_mma(cudaStream_t st, const PackedArgs& a, int n_items);
template <typename T> int packed_dkv_mma(cudaStream_t st, const PackedArgs& a, int n_items);
// items: tiles of 128 rows of both sides
template <typename T> int packed_delta(cudaStream_t st, const PackedArgs& a, const int4* items_q, int n_q, const int4* items_kv, int n_kv);
// joins of the pieces' shares (a.pieces of the forward kernel; of dq, of dk and dv)
template <typename T> int packed_join(cudaStream_t st, const PackedArgs& a);
template <typename T> int packed_sum(cudaStream_t st, const PackedArgs& a, int pieces_q, int pieces_kv);

// Kernels on the tensor cores: tiles of 128 rows, two of them side by side in the forward kernel.  float32 (d <= 64) runs on operands that
// are split into three bfloat16 terms ahead (packed_split_bytes of workspace).
// Whether the forward kernel's CTAs have one tile of 128 rows and half of an SM, or two and all of it.  About 8,200 rows in structures of up to L, one
// tile / two, us: 8 heads x 128, L = 128 23 / 29, 512 37 / 39, 1,024 54 / 51, 16,001 rows to 8,192 777 / 680 (keys and values come in
// twice as often, through half the buffers); 8 x 64 512 29 / 34, 2,048 64 / 75, 9 heads of 8,192 rows 254 / 268; float32 4 x 32, 256
// 31 / 34, 1,024 45 / 53, 5,000 rows 120 / 115.
inline bool packed_one_tile(bool f32, int d, int longest_kv) { return f32 ? d <= 32 && longest_kv < 2048 : d <= 64 || longest_kv < 800; }
struct PackedPieces { int forward = 1, dq = 1, dkv = 1; };
template <typename T> int packed_forward_tc(cudaStream_t st, PackedArgs a, int n_items, const PackedPieces& pieces, void* workspace);
template <typename T>
int packed_reverse_tc(cudaStream_t st, PackedArgs a, const int4* items_q, int n_q, const int4* items_kv, int n_kv, const PackedPieces& pieces, void* workspace);
inline int packed_split_width(int d) { return d <= 32 ? 32 : 64; }
inline int64_t packed_split_bytes(int64_t rows_q, int64_t rows_kv, int hq, int hk, int d, bool reverse) {
  return ((reverse ? 2 : 1) * rows_q * hq + 2 * rows_kv * hk) * 3 * packed_split_width(d) * 2;
}
int packed_error_word(int** word);

// shares of the pieces, behind the split operands
inline int64_t packed_share_bytes(const PackedPieces& p, int64_t rows_q, int64_t rows_kv, int hq, int hk, int d, bool reverse) {
  if (!reverse) return p.forward > 1 ? p.forward * rows_q * hq * (d + 2) * 4 : 0;
  return (p.dq > 1 ? p.dq * rows_q * hq * d * 4 : 0) + (p.dkv > 1 ? 2 * p.dkv * rows_kv * hk * d * 4 : 0);
}

inline int packed_padded(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }

}  // namespace so3lr
