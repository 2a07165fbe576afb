// Attention inside the structures of a packed batch: the work items of a batch's layout, and which kernels a call runs.
#include "packed_attention.h"

#include "../../include/so3lr_b200.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <exception>
#include <vector>

#include "kernels.h"

namespace so3lr {
namespace {

// The image of a layout (int32): a header, the offsets of both sides, and tables of work items {structure, tile, first, last}.
// Tables of query tiles: 64 rows (warp-level kernels), 128 and 256 (tensor cores, reverse and forward); of key tiles: 64 and 128; of both
// with 16 rows where no structure has more than kShortRows.
enum Head : int { kMagicAt, kN, kCausal, kRowsQ, kRowsKv, kMaxQ, kStartQ, kStartKv, kItemsQ, kNItemsQ, kItemsKv, kNItemsKv, kItemsSplit, kNItemsSplit,
                  kSplitFirst, kCombine, kTotal, kItemsQ128, kNItemsQ128, kItemsQ256, kNItemsQ256, kItemsKv128, kNItemsKv128, kMaxKv,
                  // tiles of 64 and of 128 that the items of a table walk over in all
                  kWalkQ, kWalkKv, kWalkQ128, kWalkQ256, kWalkKv128,
                  kItemsQ16, kNItemsQ16, kItemsKv16, kNItemsKv16, kHeadInts = 48 };
constexpr int kMagic = 0x53334c50;
constexpr int kTables = 7, kTileRows[kTables] = {kPackTile, kPackTile, 128, 256, 128, 16, 16};
constexpr int kTableAt[kTables] = {kItemsQ, kItemsKv, kItemsQ128, kItemsQ256, kItemsKv128, kItemsQ16, kItemsKv16};
constexpr bool kOfKeys[kTables] = {false, true, false, false, true, false, true};
constexpr int kShortRows = 48;

int64_t align4(int64_t x) { return (x + 3) & ~3LL; }

// Stretches of the keys in the form for few queries.  A stretch of 512 keys is long enough that its CTA's start costs little; with few
// keys in all, shorter ones give every SM two.
int split_length(int64_t keys) {
  const int64_t want = (keys + 295) / 296;
  return (int)std::min<int64_t>(512, std::max<int64_t>(64, (want + 63) / 64 * 64));
}

struct Counts { int64_t items[kTables] = {}, split = 0, total = 0; };

bool valid(int n, const int32_t* sq, const int32_t* sk) {
  if (n < 0 || !sq || !sk || sq[0] != 0 || sk[0] != 0) return false;
  for (int i = 0; i < n; ++i) if (sq[i + 1] < sq[i] || sk[i + 1] < sk[i]) return false;
  return true;
}

bool all_short(int n, const int32_t* sq, const int32_t* sk) {
  for (int i = 0; i < n; ++i) if (sq[i + 1] - sq[i] > kShortRows || sk[i + 1] - sk[i] > kShortRows) return false;
  return true;
}

Counts count(int n, const int32_t* sq, const int32_t* sk) {
  Counts c;
  const int chunk = split_length(sk[n]);
  for (int i = 0; i < n; ++i) {
    const int64_t lq = sq[i + 1] - sq[i], lk = sk[i + 1] - sk[i];
    for (int t = 0; t < kTables; ++t) c.items[t] += ((kOfKeys[t] ? lk : lq) + kTileRows[t] - 1) / kTileRows[t];
    if (lq > 0) c.split += std::max<int64_t>(1, (lk + chunk - 1) / chunk);
  }
  if (!all_short(n, sq, sk)) c.items[5] = c.items[6] = 0;
  c.total = kHeadInts + 3 * align4(n + 1) + 4 * c.split;
  for (int t = 0; t < kTables; ++t) c.total += 4 * c.items[t];
  return c;
}

struct Item { int32_t s, tile, first, last; };

void put(int32_t* at, std::vector<Item>& items) {
  // the longest first, so that what is left at the end is short
  std::stable_sort(items.begin(), items.end(), [](const Item& a, const Item& b) { return a.last - a.first > b.last - b.first; });
  for (size_t i = 0; i < items.size(); ++i) { at[4 * i] = items[i].s; at[4 * i + 1] = items[i].tile; at[4 * i + 2] = items[i].first; at[4 * i + 3] = items[i].last; }
}

void build_image(int n, const int32_t* sq, const int32_t* sk, bool causal, int32_t* im) {
  const Counts c = count(n, sq, sk);
  std::fill(im, im + c.total, 0);
  im[kMagicAt] = kMagic; im[kN] = n; im[kCausal] = causal; im[kRowsQ] = sq[n]; im[kRowsKv] = sk[n]; im[kTotal] = (int32_t)c.total;
  int64_t at = kHeadInts;
  auto place = [&](int field, int64_t ints) { im[field] = (int32_t)at; at += ints; };
  place(kStartQ, align4(n + 1)); place(kStartKv, align4(n + 1)); place(kSplitFirst, align4(n + 1));
  for (int t = 0; t < kTables; ++t) { place(kTableAt[t], 4 * c.items[t]); im[kTableAt[t] + 1] = (int32_t)c.items[t]; }
  place(kItemsSplit, 4 * c.split); im[kNItemsSplit] = (int32_t)c.split;
  std::copy(sq, sq + n + 1, im + im[kStartQ]);
  std::copy(sk, sk + n + 1, im + im[kStartKv]);
  std::vector<Item> items;
  for (int t = 0; t < kTables; ++t) {
    const int64_t rows = kTileRows[t];
    if (c.items[t] == 0) continue;
    items.clear();
    items.reserve(c.items[t]);
    for (int s = 0; s < n; ++s) {
      const int64_t lq = sq[s + 1] - sq[s], lk = sk[s + 1] - sk[s], off = lk - lq;
      if (!kOfKeys[t]) {      // the keys that a tile's last row sees
        for (int64_t i = 0; i * rows < lq; ++i)
          items.push_back({s, (int32_t)i, 0, (int32_t)(causal ? std::min(lk, std::max<int64_t>(0, std::min(lq, (i + 1) * rows) + off)) : lk)});
      } else {                // the queries from the first one on that sees the tile's first key
        for (int64_t i = 0; i * rows < lk; ++i)
          items.push_back({s, (int32_t)i, (int32_t)(causal ? std::min(lq, std::max<int64_t>(0, i * rows - off)) : 0), (int32_t)lq});
      }
    }
    put(im + im[kTableAt[t]], items);
    int64_t walk = 0;
    for (const Item& i : items) walk += t < 2 ? (i.last - i.first + 63) / 64 : (i.last - i.first + 127) / 128;
    if (t < 5) im[kWalkQ + t] = (int32_t)std::min<int64_t>(walk, 0x7fffffff);
  }
  const int chunk = split_length(sk[n]);
  int32_t* split = im + im[kItemsSplit];
  int k = 0;
  for (int s = 0; s < n; ++s) {
    const int lq = sq[s + 1] - sq[s], lk = sk[s + 1] - sk[s];
    im[kMaxQ] = std::max(im[kMaxQ], lq); im[kMaxKv] = std::max(im[kMaxKv], lk);
    im[im[kSplitFirst] + s] = k;
    if (lq == 0) continue;
    const int pieces = (int)std::max<int64_t>(1, ((int64_t)lk + chunk - 1) / chunk);
    if (pieces > 1) im[kCombine] = 1;
    for (int p = 0; p < pieces; ++p, ++k) {
      split[4 * k] = s; split[4 * k + 1] = pieces;
      split[4 * k + 2] = (int32_t)((int64_t)p * chunk); split[4 * k + 3] = (int32_t)std::min<int64_t>(lk, (p + 1LL) * chunk);
    }
  }
  im[im[kSplitFirst] + n] = k;
}

bool rows_ok(const so3lr_b200_rows* r, int type) {
  const long long unit = type == kF32 ? 4 : 8;
  return r && r->data && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->row_stride % unit == 0 && r->head_stride % unit == 0;
}
Rows rows_of(const so3lr_b200_rows* r) { return {r->data, r->row_stride, r->head_stride}; }

bool shape_ok(const int32_t* im, const so3lr_b200_attention_shape* a) {
  return im && im[kMagicAt] == kMagic && a && a->type >= 0 && a->type <= 2 && a->heads_q > 0 && a->heads_kv > 0 && a->heads_q % a->heads_kv == 0 &&
         a->heads_q <= 65535 && a->d >= 16 && a->d <= 128 && a->d % 16 == 0 && a->rows_q >= im[kRowsQ] && a->rows_q < 0x7fffffff && a->rows_kv >= im[kRowsKv] && a->rows_kv < 0x7fffffff &&
         a->scale > 0.f && std::isfinite(a->scale);
}

// Batches of structures this short take warp-level CTAs of one warp and 16 rows.  Forward and backward, 16 rows / 64 rows, us: 512 structures of 10
// to 40, float32 4 heads x 32, 74 / 86; 160 of 28 to 56, bfloat16 8 x 32 41 / 39; 300 of 10 to 32, bfloat16 8 x 64, 48 / 74, 160 of 28 to
// 56 67 / 58; 600 of up to 17, bfloat16 32 x 96, 290 / 591; 316 of 17 to 32, float32 2 x 128, 144 / 132.
int short_rows(int d) { return d <= 32 ? kShortRows : d <= 64 ? 40 : 24; }

PackedArgs common(const int32_t* im, const int32_t* dev, const so3lr_b200_attention_shape* a) {
  PackedArgs p;
  p.start_q = dev + im[kStartQ]; p.start_kv = dev + im[kStartKv]; p.split_first = dev + im[kSplitFirst];
  p.rows = im[kRowsQ]; p.rows_kv = im[kRowsKv]; p.longest_kv = im[kMaxKv]; p.structures = im[kN];
  if (std::max(im[kMaxQ], im[kMaxKv]) <= short_rows(a->d)) p.tile_rows = 16;
  p.stages = im[kMaxKv] <= (p.tile_rows == 16 || (a->type == kF32 && a->d > 64) ? 32 : 64) ? 1 : 2;
  p.rev_stages = im[kMaxKv] <= 32 && im[kMaxQ] <= 32 && a->heads_q == a->heads_kv ? 1 : 2;
  p.nq = (int)a->rows_q; p.nkv = (int)a->rows_kv; p.hq = a->heads_q; p.hk = a->heads_kv; p.group = a->heads_q / a->heads_kv; p.d = a->d; p.causal = im[kCausal];
  p.scale = a->scale; p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
  return p;
}

int64_t part_floats(const int32_t* im, const so3lr_b200_attention_shape* a) {
  return (int64_t)im[kNItemsSplit] * a->heads_kv * im[kMaxQ] * (a->heads_q / a->heads_kv) * packed_padded(a->d);
}

// Batches whose longest structure has this many rows on both sides go to the tensor-core kernels, whose tiles hold 128 rows and whose CTAs
// take some us to start and end.  Tensor cores / warp-level, us, about 8,200 rows in structures between half and all of the longest, which
// has L rows (float32 above 64 values has warp-level kernels only):
//   forward   16-bit, 4 heads x 32:  L = 512 17.9 / 16.4,  640 19.8 / 18.5                  float32, 4 x 32:  192 24.8 / 22.3,  256 26.8 / 26.2
//             16-bit, 8 x 64:        L = 192 23.0 / 22.3,  224 22.8 / 24.8                   float32, 8 x 64:  192 82 / 79,  224 80 / 92
//             16-bit, 8 x 128:       L =  64 28.2 / 28.4,   80 30.5 / 40.0
//   reverse   16-bit, 4 x 32:        L = 320 39 / 37,  384 37 / 40                           float32, 4 x 32:   80 60 / 51,  96 52 / 53
//             16-bit, 8 x 64:        L =  80 65 / 57,   96 57 / 61                           float32, 8 x 64:   64 210 / 142,  80 177 / 190
//             16-bit, 8 x 128:       L =  64 109 / 100,  80 96 / 121
int tensor_core_rows(int type, int d, bool reverse) {
  if (type == kF32) return d <= 32 ? (reverse ? 96 : 224) : d <= 64 ? (reverse ? 80 : 200) : 0x7fffffff;
  return d <= 32 ? (reverse ? 360 : 600) : d <= 64 ? (reverse ? 90 : 200) : 72;
}
bool on_tensor_cores(const int32_t* im, const so3lr_b200_attention_shape* a, bool reverse) {
  const int rows = tensor_core_rows(a->type, a->d, reverse);
  return im[kMaxQ] >= rows && im[kMaxKv] >= rows;
}
// Few queries: the heads of a group share one tile of rows with their token, and the keys are cut into stretches.  The keys are then
// read once per group and not once per head.
bool few_rows(const int32_t* im, const so3lr_b200_attention_shape* a) {
  return (int64_t)im[kMaxQ] * (a->heads_q / a->heads_kv) <= kPackTile;
}
// Into how many pieces the walks of a kernel's items are cut.  With few CTAs for the chip the last round of them leaves most SMs idle (160
// equal ones on 148: half of the time), so the time is that of the work on all SMs, plus half of a CTA that ends last, plus what a CTA costs
// besides its tiles (a start and an end: two tiles' time, `tile` us each), plus the shares' way through memory and the launch that joins them.
int pieces_of(int64_t items, int heads, int64_t walk, int longest, double tile, double share_bytes, int per_sm = 1) {
  if (items == 0 || walk == 0) return 1;
  const double sms = (double)sm_count() * per_sm, ctas = (double)items * heads, tiles = (double)walk * heads;
  double best = 0;
  int at = 1;
  for (int p = 1; p <= 16 && (p == 1 || longest >= 3 * p); ++p) {
    const double one = (double)longest / p + 2, rounds = std::max(1.0, ctas * p / sms);
    const double even = (tiles + 2 * ctas * p) / sms, quantised = std::ceil(ctas * p / sms) * (tiles / (ctas * p) + 2);
    const double cost = tile * std::max(even + 0.5 * one / rounds, std::min(quantised, even + one)) + (p > 1 ? 3 + p * share_bytes * 2 / 4e6 : 0);
    if (p == 1 || cost < 0.95 * best) { best = cost; at = p; }
  }
  return at;
}
// of a forward call, or of its transpose
PackedPieces pieces(const int32_t* im, const so3lr_b200_attention_shape* a, bool reverse) {
  PackedPieces p;
  if (!on_tensor_cores(im, a, reverse)) {      // 64 x 64 tiles of the warp-level kernels, two CTAs on an SM
    const int long_q = (im[kMaxQ] + 63) / 64, long_kv = (im[kMaxKv] + 63) / 64, group = a->heads_q / a->heads_kv;
    const double bytes_q = 4.0 * im[kRowsQ] * a->heads_q * a->d, bytes_kv = 4.0 * im[kRowsKv] * a->heads_kv * a->d;
    // Estimates on the low side, for a chip that is not full: with it full a tile takes a half of an SM, forward / dq / dk and dv, float32 3.5 us with 32
    // values a head, 7.0 with 64, 9 / 13 / 17 with 96, 12 / 23 / 31 with 128, bfloat16 1.4 / 1.5 / 2.3 with 32.
    const double tile = (a->type == kF32 ? 3.0 : 1.5) * (a->d <= 32 ? 0.4 : a->d <= 64 ? 0.7 : 1.3);
    if (!few_rows(im, a)) p.forward = pieces_of(im[kNItemsQ], a->heads_q, im[kWalkQ], long_kv, tile, bytes_q, 2);
    p.dq = pieces_of(im[kNItemsQ], a->heads_q, im[kWalkQ], long_kv, 1.5 * tile, bytes_q, 2);
    p.dkv = pieces_of(im[kNItemsKv], a->heads_kv, (int64_t)im[kWalkKv] * group, long_q * group, 2 * tile, 2 * bytes_kv, 2);
    return p;
  }
  const int long_q = (im[kMaxQ] + 127) / 128, long_kv = (im[kMaxKv] + 127) / 128, group = a->heads_q / a->heads_kv;
  // A tile's time, us: 256 x 128 forward (128 x 128 on half an SM up to 64 values), 128 x 128 reverse.  With the chip full and walks of 64 tiles they are
  // some tenth more: 16 bits 2.1 (1.9), 1.2 to 1.5, 1.4 to 1.8; float32 3.4, 2.1, 3.2.
  const bool f32 = a->type == kF32, wide = a->d > 64;
  const double fwd = f32 ? 3.0 : wide ? 2.1 : 1.4, dq = f32 ? 2.0 : wide ? 1.4 : 1.0, dkv = f32 ? 3.0 : wide ? 1.6 : 1.2;
  const double bytes_q = 4.0 * im[kRowsQ] * a->heads_q * a->d, bytes_kv = 4.0 * im[kRowsKv] * a->heads_kv * a->d;
  if (packed_one_tile(f32, a->d, im[kMaxKv])) p.forward = pieces_of(im[kNItemsQ128], a->heads_q, im[kWalkQ128], long_kv, fwd, bytes_q, 2);
  else p.forward = pieces_of(im[kNItemsQ256], a->heads_q, im[kWalkQ256], long_kv, fwd, bytes_q);
  p.dq = pieces_of(im[kNItemsQ128], a->heads_q, im[kWalkQ128], long_kv, dq, bytes_q);
  p.dkv = pieces_of(im[kNItemsKv128], a->heads_kv, (int64_t)im[kWalkKv128] * group, long_q * group, dkv, 2 * bytes_kv);
  return p;
}
int64_t whole_bytes(const int32_t* im, const so3lr_b200_attention_shape* a, bool reverse) {
  return (a->type == kF32 && on_tensor_cores(im, a, reverse) ? packed_split_bytes(a->rows_q, a->rows_kv, a->heads_q, a->heads_kv, a->d, reverse) : 0) +
         packed_share_bytes(pieces(im, a, reverse), a->rows_q, a->rows_kv, a->heads_q, a->heads_kv, a->d, reverse);
}
std::atomic<int> g_wait_tries{500000};      // some 4 us each: two seconds
// The device's word, and kIncomplete where an earlier call's wait has run out: told once.
int waits(PackedArgs* p) {
  const int rc = packed_error_word(&p->error);
  if (rc) return rc;
  p->wait_tries = g_wait_tries.load(std::memory_order_relaxed);
  return __atomic_load_n(p->error, __ATOMIC_RELAXED) && __atomic_exchange_n(p->error, 0, __ATOMIC_RELAXED) ? kIncomplete : kOk;
}
constexpr int64_t kQueueBytes = 16;      // behind these: PackedArgs::queue, and in the reverse pass of float16 largest and size_g
int64_t size_bytes(const int32_t* im, const so3lr_b200_attention_shape* a) {
  return a->type == kF16 && on_tensor_cores(im, a, true) ? ((int64_t)im[kN] * a->heads_kv * 2 + a->rows_q * a->heads_q) * 4 : 0;
}

const int4* table(const int32_t* im, const int32_t* dev, int field) { return reinterpret_cast<const int4*>(dev + im[field]); }

template <typename T>
int forward(cudaStream_t st, PackedArgs p, const int32_t* im, const int32_t* dev, const so3lr_b200_attention_shape* a, void* workspace) {
  if (few_rows(im, a) && (p.tile_rows != 16 || im[kMaxQ] * p.group <= 16)) {
    p.items = table(im, dev, kItemsSplit);
    p.part_rows = im[kMaxQ] * p.group;
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + part_floats(im, a));
    return packed_forward_split<T>(st, p, im[kNItemsSplit], im[kN], im[kCombine]);
  }
  if (on_tensor_cores(im, a, false)) {
    const bool one = packed_one_tile(a->type == kF32, a->d, im[kMaxKv]);
    p.items = table(im, dev, one ? kItemsQ128 : kItemsQ256);
    p.queue = reinterpret_cast<int*>(static_cast<char*>(workspace) + whole_bytes(im, a, false));
    return packed_forward_tc<T>(st, p, im[one ? kNItemsQ128 : kNItemsQ256], pieces(im, a, false), workspace);
  }
  const bool small = p.tile_rows == 16;
  p.items = table(im, dev, small ? kItemsQ16 : kItemsQ);
  p.pieces = pieces(im, a, false).forward;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)p.pieces * p.nq * p.hq * p.d);
  const int rc = packed_forward_mma<T>(st, p, im[small ? kNItemsQ16 : kNItemsQ]);
  return rc || p.pieces == 1 ? rc : packed_join<T>(st, p);
}

template <typename T>
int reverse(cudaStream_t st, PackedArgs p, const int32_t* im, const int32_t* dev, const so3lr_b200_attention_shape* a, void* workspace) {
  char* behind = static_cast<char*>(workspace) + whole_bytes(im, a, true);
  if (on_tensor_cores(im, a, true)) { p.queue = reinterpret_cast<int*>(behind); behind += kQueueBytes; }
  if (size_bytes(im, a)) {
    p.largest = reinterpret_cast<unsigned*>(behind);
    p.size_g = reinterpret_cast<float*>(p.largest + (int64_t)im[kN] * p.hk * 2);
  }
  int rc = packed_delta<T>(st, p, table(im, dev, kItemsQ128), im[kNItemsQ128], table(im, dev, kItemsKv128), im[kNItemsKv128]);
  if (rc) return rc;
  if (on_tensor_cores(im, a, true))
    return packed_reverse_tc<T>(st, p, table(im, dev, kItemsQ128), im[kNItemsQ128], table(im, dev, kItemsKv128), im[kNItemsKv128], pieces(im, a, true), workspace);
  const PackedPieces n = pieces(im, a, true);
  const int64_t stride_q = (int64_t)p.nq * p.hq * p.d, stride_kv = (int64_t)p.nkv * p.hk * p.d;
  float* share = static_cast<float*>(workspace);
  if (n.dq > 1) { p.share[0] = share; share += n.dq * stride_q; }
  if (n.dkv > 1) { p.share[1] = share; p.share[2] = share + n.dkv * stride_kv; }
  const bool small = p.tile_rows == 16;
  p.items = table(im, dev, small ? kItemsQ16 : kItemsQ);
  p.pieces = n.dq;
  if (im[kNItemsQ]) rc = packed_dq_mma<T>(st, p, im[small ? kNItemsQ16 : kNItemsQ]);
  if (rc) return rc;
  p.items = table(im, dev, small ? kItemsKv16 : kItemsKv);
  p.pieces = n.dkv;
  if (im[kNItemsKv]) rc = packed_dkv_mma<T>(st, p, im[small ? kNItemsKv16 : kNItemsKv]);
  return rc || (n.dq == 1 && n.dkv == 1) ? rc : packed_sum<T>(st, p, n.dq, n.dkv);
}

}  // namespace
}  // namespace so3lr

using namespace so3lr;

extern "C" {

int64_t so3lr_b200_packing_size(int n_structures, const int32_t* start_q, const int32_t* start_kv) {
  if (!valid(n_structures, start_q, start_kv)) return -1;
  const int64_t total = count(n_structures, start_q, start_kv).total;
  return total < 0x7fffffff ? total : -1;
}

int so3lr_b200_packing_build(int n_structures, const int32_t* start_q, const int32_t* start_kv, int causal, int32_t* image, int64_t capacity) {
  const int64_t need = so3lr_b200_packing_size(n_structures, start_q, start_kv);
  if (need < 0 || !image || capacity < need) return kInvalidArgument;
  try {
    build_image(n_structures, start_q, start_kv, causal != 0, image);
  } catch (const std::exception&) {
    return kTooLarge;
  }
  return kOk;
}

int64_t so3lr_b200_structure_attention_workspace(const int32_t* image, const so3lr_b200_attention_shape* a, int vjp) {
  if (!shape_ok(image, a)) return -1;
  if (vjp || !few_rows(image, a))
    return whole_bytes(image, a, vjp) + (on_tensor_cores(image, a, vjp) ? kQueueBytes : 0) + (vjp ? size_bytes(image, a) : 0);
  if (!image[kCombine]) return 0;
  return part_floats(image, a) * (int64_t)sizeof(float) + part_floats(image, a) / packed_padded(a->d) * (int64_t)sizeof(float2);
}

int so3lr_b200_structure_attention(const int32_t* image, const int32_t* image_dev, void* stream, const so3lr_b200_attention_shape* a,
                                   const so3lr_b200_rows* q, const so3lr_b200_rows* k, const so3lr_b200_rows* v, void* out, void* out_rest,
                                   float* lse, void* workspace, int64_t workspace_bytes) {
  if (!shape_ok(image, a) || !image_dev) return kInvalidArgument;
  if (image[kRowsQ] == 0) return kOk;
  if (!rows_ok(q, a->type) || (image[kRowsKv] && (!rows_ok(k, a->type) || !rows_ok(v, a->type))) || !out) return kInvalidArgument;
  const int64_t need = so3lr_b200_structure_attention_workspace(image, a, 0);
  if (need > 0 && (!workspace || workspace_bytes < need)) return kInvalidArgument;
  PackedArgs p = common(image, image_dev, a);
  const int told = waits(&p);
  if (told) return told;
  p.q = rows_of(q);
  if (image[kRowsKv]) { p.k = rows_of(k); p.v = rows_of(v); } else { p.k = p.v = p.q; }   // never read: no structure has keys
  p.out = out; p.out_rest = a->type == kF32 ? nullptr : out_rest; p.lse = lse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = a->type == kBF16 ? forward<__nv_bfloat16>(st, p, image, image_dev, a, workspace)
                 : a->type == kF16 ? forward<__half>(st, p, image, image_dev, a, workspace) : forward<float>(st, p, image, image_dev, a, workspace);
  SO3LR_CUDA_CHECK(cudaGetLastError());
  return rc;
}

int so3lr_b200_structure_attention_vjp(const int32_t* image, const int32_t* image_dev, void* stream, const so3lr_b200_attention_shape* a,
                                       const so3lr_b200_rows* q, const so3lr_b200_rows* k, const so3lr_b200_rows* v, const void* out,
                                       const void* out_rest, const float* lse, const so3lr_b200_rows* g, float* delta, void* d_q, void* d_k,
                                       void* d_v, void* workspace, int64_t workspace_bytes) {
  if (!shape_ok(image, a) || !image_dev) return kInvalidArgument;
  if (image[kRowsQ] == 0 && image[kRowsKv] == 0) return kOk;
  if ((image[kRowsQ] && (!rows_ok(q, a->type) || !rows_ok(g, a->type) || !out || !lse || !delta || !d_q)) ||
      (image[kRowsKv] && (!rows_ok(k, a->type) || !rows_ok(v, a->type) || !d_k || !d_v)))
    return kInvalidArgument;
  const int64_t need = so3lr_b200_structure_attention_workspace(image, a, 1);
  if (need > 0 && (!workspace || workspace_bytes < need)) return kInvalidArgument;
  PackedArgs p = common(image, image_dev, a);
  const int told = waits(&p);
  if (told) return told;
  if (image[kRowsQ]) { p.q = rows_of(q); p.g = rows_of(g); }
  if (image[kRowsKv]) { p.k = rows_of(k); p.v = rows_of(v); }
  if (!image[kRowsQ]) p.q = p.g = p.k;      // never read: one side has no rows
  if (!image[kRowsKv]) p.k = p.v = p.q;
  p.o.p = out; p.out_rest = const_cast<void*>(a->type == kF32 ? nullptr : out_rest); p.lse = const_cast<float*>(lse); p.delta = delta; p.dq = d_q; p.dk = d_k; p.dv = d_v;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = a->type == kBF16 ? reverse<__nv_bfloat16>(st, p, image, image_dev, a, workspace)
                 : a->type == kF16 ? reverse<__half>(st, p, image, image_dev, a, workspace) : reverse<float>(st, p, image, image_dev, a, workspace);
  SO3LR_CUDA_CHECK(cudaGetLastError());
  return rc;
}

int so3lr_b200_structure_attention_error(int* out) {
  if (!out) return kInvalidArgument;
  int* word = nullptr;
  const int rc = packed_error_word(&word);
  if (rc) return rc;
  SO3LR_CUDA_CHECK(cudaDeviceSynchronize());
  *out = __atomic_exchange_n(word, 0, __ATOMIC_RELAXED);
  return kOk;
}

int so3lr_b200_host_wait_tries(int tries) { return g_wait_tries.exchange(tries); }

}  // extern "C"
