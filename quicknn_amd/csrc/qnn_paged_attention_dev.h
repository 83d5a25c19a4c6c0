// qnn_paged_attention_dev.h -- attention of a batch of sequences over the paged
// KV cache.
//
// For a row at own position o of a sequence with P keys of a shared prefix
// before its own: out = softmax over t of score(t) times V[t], t over the
// prefix's keys and the own keys up to o, of absolute position above
// P + o - window where there is a window.  score = q . K[t] * scale, then
// softcap * tanh(score / softcap).  A row that sees no key gives zeros, and so
// does one whose scores are all minus infinity.
//
// Columns.  The rows of a sequence times the query heads of a KV head are the
// columns that read the same keys; so are the rows of all sequences of a group
// for the prefix, whose keys are read once for each tile of up to 128 of them.
// Both products run on the matrix cores transposed, S^T = K Q^T and O^T = V^T
// P^T, 32 columns by 32 keys: a lane's results then belong to one column, its
// running maximum, sum and rescaling are in-lane (one exchange of the two
// half-waves), and the weights are, as they stand in its registers, the operand
// of the second product.  Pages hold K and V in operand order, so nothing is
// rearranged.
//
// Arithmetic.  A BF16 cache multiplies on v_mfma_f32_32x32x16_bf16, three
// products each: q and the weights are split into three bf16 planes by
// truncation, 8 bits each, which is all of an fp32 value; K and V are exact as
// they are.  An F32 cache multiplies on v_mfma_f32_32x32x2_f32.  Maxima, sums
// and outputs are fp32.  Weights are powers of two of scores times log2(e),
// which is in q (or, with a cap, in the factor behind the tanh).
//
// Work.  The keys of a tile of columns and a KV head are an item, counted in
// units of 32.  Items lie on one line, cut into equal shares, one per
// workgroup, whatever the lengths of the sequences are: every workgroup adds
// up the lengths (they are on the device) and finds its share.  A share's part
// of an item leaves its maximum, sum and output for k_paged_join, unless it is
// the whole item and there is no prefix.  Up to 32 columns (`narrow`: single
// tokens) the four waves of a workgroup take every fourth unit; more (`wide`)
// are tiles of 128 columns, 32 per wave, with the units staged in LDS.
//
// What bounds it (32 query heads on 8, 128 channels, BF16, per call).  Single
// tokens: memory, forty sequences up to 8k keys (736 MB) 124 us, 6.3 TB/s in the
// main kernel, matrix cores 14 % busy; one token at 4k keys 15 us, a chain of
// latencies (share 3 us, table, K, V, join of the waves, second launch).  Many
// columns: the matrix cores with their three products, 1000 rows over 8000 keys
// 343 us (369 GFLOP of products, 1.08 PFLOP/s; a large library product reaches
// 1.14 on this card).
//
// Infinities and NaN.  A plane or weight of zero times an infinity would be
// NaN, also in keys that a column does not see.  So a part with a NaN in its
// result is computed again, column by column, in plain fp32 (slow_column),
// which gives what the formula gives.
#pragma once
#include <cmath>

#include "qnn_exchange.h"
#include "qnn_paged_dev.h"
#include "qnn_topk_dev.h"

namespace qnn {
namespace {

constexpr int kThreads = 256;
constexpr int kNarrow = 32, kWide = 128;  // columns of a tile, at most
constexpr int kUnit = 32;                 // keys
constexpr float kLog2e = 1.4426950408889634f;

// An item that a worker began and did not end: n parts, from this worker's on.
struct Split {
  int first, h, c0, cols, n;  // first row of the owner; KV head, first column and columns of the tile
};
struct Line;

struct Args {
  PagedAttn a;
  int group, owners, workers;        // query heads per KV head; sequences (and groups, with prefixes)
  int narrow;                        // columns up to which an owner is a narrow tile: 16 or 32
  float qmul, smul;                  // scores are q qmul . K; with a cap smul tanh of that
  Line *head[2];                     // of the narrow and wide tiles (with prefixes)
  int *table[2];                     // where a tile begins on its line (with prefixes)
  Split *splits[2];                  // per worker (without)
  float *parts[2];                   // of split items, [2 workers][columns][dim + 4]: output, maximum, sum
  int cols[2];                       // columns of a part
  float *whole;                      // of whole items (with prefixes), [own, prefix][KV head][rows x group][dim + 4]
  int prefix_tiles;                  // id of the first wide tile of the prefixes
  int *first_keys;                   // per group: the first prefix key that any row sees (with prefixes and a window)
};

__device__ __forceinline__ int row_sequence(const PagedBatch &b, int row) {
  if (!b.starts) return row;
  int lo = 0, hi = b.sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (dev::first_row(b, mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// (find_share reads every owner and reports what is out of range; elsewhere
// values are only brought into it.)
// A set of columns over the same keys: sequence o's rows over its own keys, or
// (o >= sequences) a group's rows over its prefix.
struct Owner {
  const int *table;
  int prefix_group;  // -1: own keys
  int first, end;    // rows
  int keys, prefix;  // keys of this owner; of the group's prefix
  int low;           // prefix with a window: the first key that any row sees
  int cols;
};

template <bool REPORT = false>
__device__ __forceinline__ Owner owner_of(const Args &g, int o) {
  const PagedBatch &b = g.a.b;
  Owner w;
  w.low = 0;
  if (o < b.sequences) {
    w.prefix_group = -1;
    dev::row_range<REPORT>(b, o, w.first, w.end);
    w.keys = dev::own_length<REPORT>(b, o);
    w.prefix = dev::prefix_length<REPORT>(b, o / b.share);
    w.table = b.tables + size_t(o) * b.table_pages;
  } else {
    const int p = o - b.sequences;
    w.prefix_group = p;
    w.first = dev::first_row(b, p * b.share);
    w.end = max(w.first, dev::first_row(b, (p + 1) * b.share));
    w.keys = w.prefix = dev::prefix_length<REPORT>(b, p);
    w.table = b.prefix_tables + size_t(p) * b.prefix_pages;
    if (g.a.window > 0 && w.keys > 0) w.low = g.first_keys[p];
  }
  w.cols = (w.end - w.first) * g.group;
  return w;
}

// Keys [low, high) that any column of the tile from column c0 may see.
template <int CT>
__device__ __forceinline__ void tile_keys(const Args &g, const Owner &w, int c0, int &low, int &high) {
  low = w.low;
  high = w.keys;
  if (w.prefix_group < 0) {
    const int at = w.keys - w.end + w.first;  // own position of the first row
    high = max(0, at + (min(c0 + CT, w.cols) - 1) / g.group + 1);
    if (g.a.window > 0) low = max(0, at + c0 / g.group - g.a.window + 1);
  }
}
template <int CT>
__device__ __forceinline__ int tile_units(const Args &g, const Owner &w, int tile) {
  int low, high;
  tile_keys<CT>(g, w, tile * CT, low, high);
  return high > low ? (high + kUnit - 1) / kUnit - low / kUnit : 0;
}
// Whether the tiles of this owner are of CT columns, and how many.
template <int CT>
__device__ __forceinline__ int owner_tiles(const Args &g, const Owner &w) {
  if (CT == kNarrow) return w.cols > 0 && w.cols <= g.narrow;
  return w.cols > g.narrow ? (w.cols + CT - 1) / CT : 0;
}
// Tiles have ids that ascend along the line: narrow ones their owner, wide
// ones the 128-column block of their owner's first column and the owner.
template <int CT>
__device__ __forceinline__ int first_tile_id(const Args &g, const Owner &w, int o) {
  if (CT == kNarrow) return o;
  const int block = int(int64_t(w.first) * g.group / CT);
  return w.prefix_group < 0 ? block + o : g.prefix_tiles + block + w.prefix_group;
}

// What a column sees of an owner's keys: [low, high).
__device__ __forceinline__ void column_keys(const Args &g, const Owner &w, int c, int &row, int &low, int &high) {
  const PagedBatch &b = g.a.b;
  row = w.first + c / g.group;
  int at;  // in this owner's keys
  if (w.prefix_group < 0) {
    at = w.keys - w.end + row;
  } else {
    const int s = row_sequence(b, row);
    int first, end;
    dev::row_range<false>(b, s, first, end);
    at = w.prefix + dev::own_length<false>(b, s) - end + row;
  }
  high = min(max(at + 1, 0), w.keys);
  low = g.a.window > 0 ? max(0, at - g.a.window + 1) : 0;
}

struct Piece {
  int h, c0, cols;        // KV head, first column of the tile, its columns
  int unit0, units;       // key units, from key 0 of the owner
  int low, high;          // keys that any column sees
  float *part;            // where the result goes; null: to the output
};

// The place of a column in q and out.
__device__ __forceinline__ size_t column_place(const Args &g, const Owner &w, const Piece &p, int c) {
  const int col = p.c0 + c, row = w.first + col / g.group;
  return (size_t(row) * g.a.heads + p.h * g.group + col % g.group) * g.a.c.dim;
}

template <int E>
__device__ __forceinline__ float element(const void *p, size_t i) {
  if constexpr (E == 8) return __uint_as_float(uint32_t(static_cast<const uint16_t *>(p)[i]) << 16);
  else return static_cast<const float *>(p)[i];
}

// One column of a piece by the whole workgroup in plain fp32, a key per
// thread, then a channel per thread.  Not inlined: it would take registers
// from the loops of its callers.
template <int E>
__device__ __attribute__((noinline)) void slow_column(const Args *args, const Owner *owner, const Piece *piece, int c,
                                                      float *lds) {
  const Args &g = *args;
  const Owner &w = *owner;
  const Piece &p = *piece;
  const PagedCache &cache = g.a.c;
  const int dim = cache.dim, tid = threadIdx.x, run = cache.page_size * dim;
  float *qs = lds, *ps = lds + 256, *red = lds + 512;
  const bool on = tid < kThreads;  // the first four waves
  const size_t place = column_place(g, w, p, c);
  int row, low, high;
  column_keys(g, w, p.c0 + c, row, low, high);
  const int from = max(low, p.unit0 * kUnit), to = min(high, (p.unit0 + p.units) * kUnit);
  __syncthreads();
  if (on && tid < dim) qs[tid] = g.a.q[place + tid] * g.qmul;
  auto page_of = [&](int t) {
    return max(dev::checked_page(w.table[t >> g.a.b.page_shift], g.a.b), 0) * size_t(2 * cache.kv_heads) * run;
  };
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int t0 = from; t0 < to; t0 += kThreads) {
    const int t = t0 + tid, n = min(kThreads, to - t0);
    __syncthreads();
    float sc = -INFINITY;
    if (on && t < to) {
      const size_t k = page_of(t) + size_t(p.h) * run;
      float dot = 0.0f;
      for (int d = 0; d < dim; ++d)
        dot += qs[d] * element<E>(cache.pages, k + dev::key_place<E>(t & (cache.page_size - 1), d, dim));
      sc = g.a.softcap > 0.0f ? g.smul * tanh20(dot) : dot;
    }
    const float mx = dev::wave_max_xor(sc);
    if (on && (tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float keep = m_new == -INFINITY ? 1.0f : exp2f(m - m_new);
    if (on) ps[tid] = t < to && (m_new > -INFINITY || sc != sc) ? exp2f(sc - m_new) : 0.0f;
    __syncthreads();
    l *= keep;
    acc *= keep;
    for (int j = 0; j < n; ++j) {
      l += ps[j];
      if (tid < dim)
        acc += ps[j] * element<E>(cache.pages, page_of(t0 + j) + size_t(cache.kv_heads + p.h) * run +
                                                   dev::value_place<E>((t0 + j) & (cache.page_size - 1), tid, dim));
    }
    m = m_new;
  }
  if (p.part) {
    float *part = p.part + size_t(c) * (dim + 4);
    if (tid == 0) {
      part[dim] = m;
      part[dim + 1] = l;
    }
    if (tid < dim) part[tid] = acc;
  } else if (tid < dim) {
    g.a.out[place + tid] = l > 0.0f || l != l ? acc / l : 0.0f;
  }
}

// ---------------------------------------------------------------------------
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x4 load16(const void *base, size_t bytes) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(base) + bytes));
}

// The key (of a unit) of row m of the score tile: what pairs a lane's weights
// with the tokens of a piece of values.
template <bool BF>
__device__ __forceinline__ constexpr int tile_key(int m) {
  if (!BF) return m;
  return (m & 7) | (m & 8) << 1 | (m & 16) >> 1;
}

// Eight fp32 values into three bf16 planes by truncation.  Each plane holds
// the next 8 bits of the value, so their sum is the value; an infinity leaves a
// NaN in the others, and its column to slow_column.
__device__ __forceinline__ void planes3(const float (&v)[8], u32x4 &hi, u32x4 &mid, u32x4 &lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a0 = __float_as_uint(v[2 * i]), a1 = __float_as_uint(v[2 * i + 1]);
    const float r0 = v[2 * i] - __uint_as_float(a0 & 0xffff0000u), r1 = v[2 * i + 1] - __uint_as_float(a1 & 0xffff0000u);
    const uint32_t b0 = __float_as_uint(r0), b1 = __float_as_uint(r1);
    const float s0 = r0 - __uint_as_float(b0 & 0xffff0000u), s1 = r1 - __uint_as_float(b1 & 0xffff0000u);
    hi[i] = __builtin_amdgcn_perm(a1, a0, 0x07060302u);
    mid[i] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
    lo[i] = __builtin_amdgcn_perm(__float_as_uint(s1), __float_as_uint(s0), 0x07060302u);
  }
}

__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma4(u32x4 a, u32x4 b, f32x16 c) {  // four steps of two keys or channels
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  return c;
}

// NK: channels / 16.
template <int NK, bool BF>
struct Shape {
  static constexpr int ND = (NK + 1) / 2;            // 32-channel tiles of the output
  static constexpr int KP = BF ? NK : 2 * NK;        // 16-byte pieces of a key per half-wave
  static constexpr int VP = BF ? 2 : 4;              // pieces of a unit's values per channel and half-wave
  static constexpr int E = BF ? 8 : 4;
  static constexpr int QL = BF ? 3 : 1;              // planes of q
  static constexpr int Q_BYTES = QL * KP * 64 * 16;  // fragments of 32 columns
};

// One column's running state (both half-waves of a column hold the same
// maximum, each its own keys' sum) and output tile.
template <int ND>
struct Running {
  float m, l;
  f32x16 o[ND];
};

// Scores (of tile_key order) to weights; updates maximum, sum and output
// scale.  `base`: the unit's first key.
template <bool BF, int ND>
__device__ __forceinline__ void soften(const Args &g, Running<ND> &r, f32x16 &s, int base, int low, int high, int half) {
  if (g.a.softcap > 0.0f)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = g.smul * tanh20(s[i]);
  if (__ballot(base < low || base + kUnit > high))  // some column does not see all of the unit
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = base + tile_key<BF>(8 * (i >> 2) + (i & 3)) + 4 * half;
      if (key < low || key >= high) s[i] = -INFINITY;
    }
  float mx = s[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
  mx = fmaxf(mx, dev::xor_lanes<32>(mx));
  // The maximum only moves when it would let weights pass 2^8: sums and
  // outputs are relative to it, whatever it is.
  if (__ballot(mx > r.m + 8.0f || (r.m == -INFINITY && mx > r.m))) {
    const float m_new = fmaxf(r.m, mx), keep = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(r.m - m_new);
    r.m = m_new;
    r.l *= keep;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[t][i] *= keep;
  }
  const float m_sub = r.m == -INFINITY ? 0.0f : r.m;  // nothing seen yet: every weight is 2^-inf = 0
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i] = __builtin_amdgcn_exp2f(s[i] - m_sub);
    r.l += s[i];
  }
}

// The line of units.  Items follow each other, tile by tile, KV head by KV
// head; workgroup x has [x share, (x + 1) share).  A part costs a workgroup its
// set-up and end, about what kItemCost units take, so an item occupies that
// much more than its units (512 workgroups, 256 items of one unit behind 32 of
// 375: 150 us without, as the last workgroups had 24 items each).  Or, aligned,
// every item starts at a multiple of the share and no workgroup has parts of
// two; that is taken where its largest part is not much longer.  At least
// kShareMin units, one per wave.  Sequences and lengths are on the device, so
// each workgroup adds them up.
constexpr int kShareMin = 4;
constexpr int kLineMax = 1 << 28;  // units of a call, at most (the host checks)
template <int CT>
constexpr int kItemCost = CT == kWide ? 4 : 8;
struct Line {
  int share, aligned;
};
template <int CT>
__device__ __forceinline__ int padded(const Line &l, int units) {
  return l.aligned ? int((unsigned(units) + unsigned(l.share) - 1) / unsigned(l.share)) * l.share
                   : units + (units ? kItemCost<CT> : 0);
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Sum of the lanes up to this one: row_shr 1, 2, 4, 8 within rows of 16 lanes,
// then row_bcast 15 and 31 across them.  (Six __shfl_up take 0.4 us.)
__device__ __forceinline__ int wave_upto(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}
__device__ __forceinline__ int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }

// Without prefixes nothing follows for tiles without keys: zeros.
template <int CT>
__device__ __attribute__((noinline)) void clear_blank_rows(const Args *args, int me) {
  const Args &g = *args;
  for (int o = me; o < g.owners; o += g.workers) {
    const Owner w = owner_of(g, o);
    for (int t = 0, n = owner_tiles<CT>(g, w); t < n; ++t) {
      if (tile_units<CT>(g, w, t)) continue;
      const int cols = min(CT, w.cols - t * CT), dim = g.a.c.dim;
      Piece p;
      p.c0 = t * CT;
      for (p.h = 0; p.h < g.a.c.kv_heads; ++p.h)
        for (int i = threadIdx.x; i < cols * dim; i += kThreads) g.a.out[column_place(g, w, p, i / dim) + i % dim] = 0.0f;
    }
  }
}

// This workgroup's share [begin, end) and where it begins.
struct Place {
  int owner, tile, unit;  // unit: within the tile's items
};
template <int CT, int NT>
__device__ __forceinline__ bool find_share(const Args &g, int me, int &begin, int &end, Line &line, Place &place, Owner &own) {
  constexpr int C = CT == kWide;
  __shared__ int sums[2][NT / 64], most[NT / 64], upto[NT / 64];
  __shared__ float roughs[NT / 64];
  __shared__ Place found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kv = g.a.c.kv_heads;
  // Up to 64 owners: every wave for itself, a lane each.  More: a run of them per thread.
  const bool few = g.owners <= 64;
  const int per = few ? 1 : (g.owners + NT - 1) / NT, o0 = min((few ? lane : tid) * per, g.owners),
            o1 = min(o0 + per, g.owners);
  // A lane's one owner is read once.
  Owner mine{};
  if (few && o0 < o1) mine = owner_of<true>(g, o0);
  auto owner = [&](int o) { return few ? mine : owner_of(g, o); };
  int units = 0, items = 0, longest = 0;
  bool blank = false;
  for (int o = o0; o < o1; ++o) {
    const Owner w = few ? mine : owner_of<true>(g, o);
    for (int t = 0, n = owner_tiles<CT>(g, w); t < n; ++t) {
      const int u = tile_units<CT>(g, w, t);
      units = min(units + kv * u, 2 * kLineMax);  // (what one owner can add is below kLineMax)
      items += u ? kv : 0;
      longest = max(longest, u);
      blank |= u == 0;
    }
  }
  // Row starts that do not ascend may give the same rows to many sequences, and
  // more units than the host allowed for: then nothing is computed.
  float rough = dev::wave_sum_xor(float(units));
  int total = last_lane(wave_upto(units)), count = last_lane(wave_upto(items));
  longest = int(dev::wave_max_u32(unsigned(longest)));
  if (!few) {
    if (lane == 0) {
      sums[0][wave] = total;
      sums[1][wave] = count;
      most[wave] = longest;
      roughs[wave] = rough;
    }
    __syncthreads();
    total = count = 0;
    rough = 0.0f;
    for (int x = 0; x < NT / 64; ++x) {
      rough += roughs[x];
      total += uniform(sums[0][x]);
      count += uniform(sums[1][x]);
      longest = max(longest, uniform(most[x]));
    }
  }
  if (!g.a.b.prefix_tables && (few ? __ballot(blank) != 0 : __syncthreads_or(blank) != 0))
    clear_blank_rows<CT>((const Args *)__builtin_amdgcn_kernarg_segment_ptr(), me);
  if (uniform(int(rough > 1.01f * kLineMax))) {
    if (tid == 0) atomicOr(g.a.b.err, kPagedErr);
    line = {kShareMin, 0};
    begin = end = 0;
    return false;
  }
  const unsigned workers = g.workers, apart = max(g.workers - count, 1);  // total / apart + count <= workers, if count is less
  const int across = int((unsigned(total + count * kItemCost<CT>) + workers - 1) / workers),
            alone = int((unsigned(total) + apart - 1) / apart);
  line.aligned = CT == kNarrow && count < g.workers && min(alone, longest) <= across + kItemCost<CT>;
  line.share = max(line.aligned ? min(alone, longest) : across, kShareMin);
  units = 0;
  for (int o = o0; o < o1; ++o) {
    const Owner w = owner(o);
    for (int t = 0, n = owner_tiles<CT>(g, w); t < n; ++t) units += kv * padded<CT>(line, tile_units<CT>(g, w, t));
  }
  int before = wave_upto(units);
  total = last_lane(before);
  before -= units;
  if (!few) {
    if (lane == 0) upto[wave] = total;
    __syncthreads();
    total = 0;
    for (int x = 0; x < NT / 64; ++x) {
      if (x < wave) before += upto[x];
      total += upto[x];
    }
  }
  total = uniform(total);
  if (me == 0 && g.a.b.prefix_tables) {  // for the join
    if (tid == 0) *g.head[C] = line;
    int at = before;
    for (int o = o0; o < o1; ++o) {
      const Owner w = owner(o);
      const int id = first_tile_id<CT>(g, w, o);
      for (int t = 0, n = owner_tiles<CT>(g, w); t < n; ++t) {
        g.table[C][id + t] = at;
        at += kv * padded<CT>(line, tile_units<CT>(g, w, t));
      }
    }
  }
  begin = line.share * me;  // at most a share past the total
  end = min(begin + line.share, total);
  if (begin >= end) return false;
  const bool here = begin >= before && begin < before + units;
  Place p{0, 0, 0};
  if (here) {
    int rest = begin - before;
    for (int o = o0; o < o1; ++o) {
      const Owner w = owner(o);
      for (int t = 0, n = owner_tiles<CT>(g, w); t < n; ++t) {
        const int u = kv * padded<CT>(line, tile_units<CT>(g, w, t));
        if (rest >= 0 && rest < u) p = {o, t, rest};
        rest -= u;
      }
    }
  }
  if (few) {
    const int from = __ffsll((unsigned long long)__ballot(here)) - 1;
    p.owner = __builtin_amdgcn_readlane(p.owner, from);
    p.tile = __builtin_amdgcn_readlane(p.tile, from);
    p.unit = __builtin_amdgcn_readlane(p.unit, from);
    auto take = [&](int x) { return __builtin_amdgcn_readlane(x, from); };
    own.prefix_group = take(mine.prefix_group);
    own.first = take(mine.first);
    own.end = take(mine.end);
    own.keys = take(mine.keys);
    own.prefix = take(mine.prefix);
    own.low = take(mine.low);
    own.cols = take(mine.cols);
    own.table = p.owner < g.a.b.sequences ? g.a.b.tables + size_t(p.owner) * g.a.b.table_pages
                                          : g.a.b.prefix_tables + size_t(p.owner - g.a.b.sequences) * g.a.b.prefix_pages;
  } else {
    if (here) found = p;
    __syncthreads();
    p = found;
  }
  place.owner = uniform(p.owner);  // the same in every lane: what follows from it stays in scalar registers
  place.tile = uniform(p.tile);
  place.unit = uniform(p.unit);
  if (!few) own = owner_of(g, place.owner);
  return true;
}

// Where the part of an item goes that worker w has.  At most two parts of a
// worker are not whole items: its first, which another worker began, and its
// last.  Whole items have places by column, and are parts only where a prefix
// and own keys are to be joined.  (A place of 128 columns for every tile that
// the host cannot rule out took 2.7 GB for 4096 beams; this 0.21 GB.)
__device__ __forceinline__ float *split_part(const Args &g, int c, int w, bool continued) {
  return g.parts[c] + (2 * int64_t(w) + !continued) * g.cols[c] * (g.a.c.dim + 4);
}
__device__ __forceinline__ float *whole_part(const Args &g, bool prefix, int h, int64_t column) {
  return g.whole + ((int64_t(prefix) * g.a.c.kv_heads + h) * g.a.b.rows * g.group + column) * (g.a.c.dim + 4);
}

// Runs body(owner, piece) for every part of this workgroup's share.
template <int CT, int NT, typename Body>
__device__ __forceinline__ void for_pieces(const Args &g, int me, Body body) {
  constexpr int C = CT == kWide;
  int at, end;
  Line line;
  Place p;
  Split split{};
  Owner w;
  if (find_share<CT, NT>(g, me, at, end, line, p, w)) {
    const int kv = g.a.c.kv_heads;
    while (at < end) {
      const int units = tile_units<CT>(g, w, p.tile), span = padded<CT>(line, units);
      if (p.tile >= owner_tiles<CT>(g, w) || p.unit >= kv * span) {
        p.unit = 0;
        if (++p.tile >= owner_tiles<CT>(g, w)) {
          if (++p.owner >= g.owners) break;
          p.tile = 0;
          w = owner_of(g, p.owner);
        }
        continue;
      }
      Piece x;
      x.h = int(unsigned(p.unit) / unsigned(span));
      const int u = p.unit - x.h * span;
      if (u >= units) {  // behind the item
        if (line.aligned) break;
        const int rest = min(span - u, end - at);
        at += rest;
        p.unit += rest;
        continue;
      }
      x.units = min(units - u, end - at);
      x.c0 = p.tile * CT;
      x.cols = min(CT, w.cols - x.c0);
      tile_keys<CT>(g, w, x.c0, x.low, x.high);
      x.unit0 = x.low / kUnit + u;
      x.part = x.units < units ? split_part(g, C, me, u > 0)
               : w.prefix      ? whole_part(g, w.prefix_group >= 0, x.h, int64_t(w.first) * g.group + x.c0)
                               : nullptr;
      if (u == 0 && x.units < units)
        split = {w.first, x.h, x.c0, x.cols, int(unsigned(at + units - 1) / unsigned(line.share)) - me + 1};
      body(w, x);
      if (line.aligned) break;
      at += x.units;
      p.unit += x.units;
    }
  }
  if (threadIdx.x == 0 && !g.a.b.prefix_tables) g.splits[C][me] = split;
}

// E channels of a column of q from channel E * piece; times the score factor,
// as operands: three planes, or the values.
template <bool BF>
struct QRaw {
  f32x4 x[BF ? 2 : 1];
  QRaw() = default;
  __device__ __forceinline__ QRaw(const float *q, int piece) {
    const f32x4 *src = reinterpret_cast<const f32x4 *>(q) + piece * (BF ? 2 : 1);
#pragma unroll
    for (int i = 0; i < (BF ? 2 : 1); ++i) x[i] = src[i];
  }
  __device__ __forceinline__ void split(const Args &g, u32x4 (&out)[BF ? 3 : 1]) const {
    if constexpr (BF) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = x[j >> 2][j & 3] * g.qmul;
      planes3(v, out[0], out[1], out[2]);
    } else {
      out[0] = __builtin_bit_cast(u32x4, x[0] * g.qmul);
    }
  }
};
template <bool BF>
__device__ __forceinline__ void load_q(const Args &g, const float *q, int piece, u32x4 (&out)[BF ? 3 : 1]) {
  QRaw<BF>(q, piece).split(g, out);
}

// The unit's weights times its values, given the value pieces of one channel
// tile.
template <bool BF>
struct Weights {
  u32x4 p[BF ? 6 : 4];
  __device__ __forceinline__ explicit Weights(const f32x16 &s) {
    if constexpr (BF) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s[8 * i + j];
        planes3(v, p[3 * i], p[3 * i + 1], p[3 * i + 2]);
      }
    } else {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[a][j] = __float_as_uint(s[4 * a + j]);
    }
  }
  template <int VP>
  __device__ __forceinline__ f32x16 times(const u32x4 (&v)[VP], f32x16 o) const {
    if constexpr (BF) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 2; j >= 0; --j) o = mfma(v[i], p[3 * i + j], o);
    } else {
#pragma unroll
      for (int a = 0; a < 4; ++a) o = mfma4(v[a], p[a], o);
    }
    return o;
  }
};

// Zeroes the elements of a value piece whose keys lie outside [low, high).
template <bool BF>
__device__ __forceinline__ void clear_outside(u32x4 &v, int base, int piece, int low, int high) {
  if constexpr (BF) {  // tokens 16 a + 4 piece + b
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = base + (i >> 1) * 16 + 4 * piece + (i & 1) * 2;
      if (key < low || key >= high) v[i] &= 0xffff0000u;
      if (key + 1 < low || key + 1 >= high) v[i] &= 0x0000ffffu;
    }
  } else {  // tokens 4 piece + b of the unit
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (base + 4 * piece + i < low || base + 4 * piece + i >= high) v[i] = 0;
  }
}

// First byte of a unit's keys of KV head h; its values are kv_heads runs on.
__device__ __forceinline__ const uint8_t *unit_base(const Args &g, const Owner &w, int h, int unit, int run,
                                                    size_t page_bytes, int token_bytes) {
  const int t = unit * kUnit;
  const int page = max(dev::checked_page(w.table[t >> g.a.b.page_shift], g.a.b), 0);
  return static_cast<const uint8_t *>(g.a.c.pages) + page * page_bytes + size_t(h) * run +
         size_t(t & (g.a.c.page_size - 1)) * token_bytes;
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16x4(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
  return c;
}

// soften for 16 columns: register 4 b + i of a lane is key 16 b + 4 quarter + i.
template <int NK>
__device__ __forceinline__ void soften16(const Args &g, float &m, float &l, f32x4 (&o)[NK], float (&s)[8], int base, int low,
                                         int high, int quarter) {
  if (g.a.softcap > 0.0f)
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = g.smul * tanh20(s[i]);
  if (__ballot(base < low || base + kUnit > high))
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = base + 16 * (i >> 2) + (i & 3) + 4 * quarter;
      if (key < low || key >= high) s[i] = -INFINITY;
    }
  float mx = s[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
  mx = fmaxf(mx, dev::xor_lanes<16>(mx));
  mx = fmaxf(mx, dev::xor_lanes<32>(mx));
  if (__ballot(mx > m + 8.0f || (m == -INFINITY && mx > m))) {
    const float m_new = fmaxf(m, mx), keep = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
    m = m_new;
    l *= keep;
#pragma unroll
    for (int t = 0; t < NK; ++t) o[t] *= keep;
  }
  const float m_sub = m == -INFINITY ? 0.0f : m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s[i] = __builtin_amdgcn_exp2f(s[i] - m_sub);
    l += s[i];
  }
}
template <bool BF>
__device__ __forceinline__ void weights16(const float (&s)[8], u32x4 (&pw)[BF ? 3 : 2]) {
  if constexpr (BF) {
    planes3(s, pw[0], pw[1], pw[2]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) pw[i >> 2][i & 3] = __float_as_uint(s[i]);
  }
}

// The four waves' results meet in LDS, relative to their common maximum.
template <int COLS>
__device__ __forceinline__ float wave_scale(const float (&wave_m)[4][COLS], int col, float m) {
  const float top = fmaxf(fmaxf(wave_m[0][col], wave_m[1][col]), fmaxf(wave_m[2][col], wave_m[3][col]));
  return top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}
template <int dim, int COLS>
__device__ __forceinline__ void join_waves(const Args &g, const Owner &w, const Piece &p, const float *os,
                                           const float (&wave_m)[4][COLS], const float (&wave_l)[4][COLS], uint32_t &redo) {
  constexpr int row = dim + 4;
  for (int i = threadIdx.x; i < p.cols * (dim / 4); i += kThreads) {
    const int c = i / (dim / 4), d = i % (dim / 4) * 4;
    f32x4 x = f32x4(0.0f);
    float l = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      x += *reinterpret_cast<const f32x4 *>(os + (v * COLS + c) * row + d);
      l += wave_l[v][c];
    }
    if (l != l || x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3]) atomicOr(&redo, 1u << c);
    if (p.part) {
      float *part = p.part + size_t(c) * row;
      if (d == 0) {
        part[dim] = fmaxf(fmaxf(wave_m[0][c], wave_m[1][c]), fmaxf(wave_m[2][c], wave_m[3][c]));
        part[dim + 1] = l;
      }
      *reinterpret_cast<f32x4 *>(part + d) = x;
    } else {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      *reinterpret_cast<f32x4 *>(g.a.out + column_place(g, w, p, c) + d) = x * inv;
    }
  }
}

// ---------------------------------------------------------------------------
// Narrow: up to 32 columns, the same for the four waves, which take every
// fourth unit.  K and V go from memory to registers in operand order; q is in
// LDS.
template <int NK, bool BF>
__device__ __forceinline__ void narrow_body(const Args &g, int me) {
  using S = Shape<NK, BF>;
  constexpr int dim = NK * 16, ND = S::ND, row = dim + 4, elem = BF ? 2 : 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ float wave_m[4][32], wave_l[4][32];
  __shared__ uint32_t redo;
  __shared__ Owner slow_owner;
  __shared__ Piece slow_piece;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
  const PagedCache &cache = g.a.c;
  const int run = cache.page_size * dim * elem;  // bytes of a head's keys in a page
  const size_t page_bytes = size_t(2) * cache.kv_heads * run;
  // Lane offsets within a unit: row `col` of the score tile, and the channel
  // (the last tile's may lie behind the last channel: any will do).
  const int key = tile_key<BF>(col);
  const uint32_t k_lane = (key >> 4) * 16 * dim * elem + (half * 16 + (key & 15)) * 16;
  const uint32_t v_lane = cache.kv_heads * run + half * dim * 16 + col * 16;
  const uint32_t v_last = NK % 2 && col >= 16 ? v_lane - 256 : v_lane;
  const u32x4 *qf = reinterpret_cast<const u32x4 *>(lds) + lane;

  for_pieces<kNarrow, kThreads>(g, me, [&](const Owner &w, const Piece &p) {
    const int last = p.unit0 + p.units;
    u32x4 kf[S::KP];
    const uint8_t *base = nullptr;
    if (p.unit0 + wave < last) {
      base = unit_base(g, w, p.h, p.unit0 + wave, run, page_bytes, dim * elem);
#pragma unroll
      for (int i = 0; i < S::KP; ++i) kf[i] = load16(base, k_lane + i * 512);
    }
    __syncthreads();  // LDS is free
    for (int i = tid; i < S::KP * 64; i += kThreads) {
      const int c = i & 31, piece = i >> 5;
      u32x4 *dst = reinterpret_cast<u32x4 *>(lds) + (piece >> 1) * 64 + (piece & 1) * 32 + c;
      u32x4 x[S::QL];
      if (c < p.cols) load_q<BF>(g, g.a.q + column_place(g, w, p, c), piece, x);
#pragma unroll
      for (int j = 0; j < S::QL; ++j) dst[j * S::KP * 64] = c < p.cols ? x[j] : u32x4(0u);
    }
    if (tid == 0) redo = 0;
    int low = 0, high = 0x7fffffff, r;
    if (col < p.cols) column_keys(g, w, col, r, low, high);
    __syncthreads();
    Running<ND> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) st.o[t] = f32x16(0.0f);
    for (int u = p.unit0 + wave; u < last; u += 4) {
      u32x4 vf[ND][S::VP];
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < S::VP; ++i) vf[t][i] = load16(base, (t == ND - 1 ? v_last : v_lane) + t * 512 + i * dim * 32);
      // One step's q on its way while another is multiplied; left alone, the
      // compiler reads all of q first and spills it.
      f32x16 s(0.0f);
      u32x4 qc[S::QL], qn[S::QL];
#pragma unroll
      for (int x = 0; x < S::QL; ++x) qc[x] = qf[x * S::KP * 64];
#pragma unroll
      for (int i = 0; i < S::KP; ++i) {
#pragma unroll
        for (int x = 0; x < S::QL; ++x) qn[x] = qf[(x * S::KP + min(i + 1, S::KP - 1)) * 64];
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BF) {
#pragma unroll
          for (int x = 2; x >= 0; --x) s = mfma(kf[i], qc[x], s);
        } else {
          s = mfma4(kf[i], qc[0], s);
        }
#pragma unroll
        for (int x = 0; x < S::QL; ++x) qc[x] = qn[x];
      }
      if (u + 4 < last) {
        base = unit_base(g, w, p.h, u + 4, run, page_bytes, dim * elem);
#pragma unroll
        for (int i = 0; i < S::KP; ++i) kf[i] = load16(base, k_lane + i * 512);
      }
      soften<BF, ND>(g, st, s, u * kUnit, low, high, half);
      if (u * kUnit < p.low || (u + 1) * kUnit > p.high)  // what is behind the last key may be anything
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
          for (int i = 0; i < S::VP; ++i) clear_outside<BF>(vf[t][i], u * kUnit, 2 * i + half, p.low, p.high);
      const Weights<BF> pw(s);
#pragma unroll
      for (int t = 0; t < ND; ++t) st.o[t] = pw.times(vf[t], st.o[t]);
    }
    st.l += dev::xor_lanes<32>(st.l);
    if (half == 0) wave_m[wave][col] = st.m;
    __syncthreads();  // q is not needed any more
    const float keep = wave_scale(wave_m, col, st.m);
    if (half == 0) wave_l[wave][col] = st.l * keep;
    float *os = reinterpret_cast<float *>(lds);
    if (col < p.cols)
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int d = t * 32 + 8 * a + 4 * half;
          if (d < dim) {
            const f32x4 x = {st.o[t][4 * a] * keep, st.o[t][4 * a + 1] * keep, st.o[t][4 * a + 2] * keep,
                             st.o[t][4 * a + 3] * keep};
            *reinterpret_cast<f32x4 *>(os + (wave * 32 + col) * row + d) = x;
          }
        }
    __syncthreads();
    join_waves<dim>(g, w, p, os, wave_m, wave_l, redo);
    __syncthreads();
    if (const uint32_t again = uniform(int(redo))) {
      slow_owner = w;
      slow_piece = p;
      __syncthreads();
      for (int c = 0; c < p.cols; ++c)
        if (again >> c & 1)
          slow_column<S::E>((const Args *)__builtin_amdgcn_kernarg_segment_ptr(), &slow_owner, &slow_piece, c,
                            reinterpret_cast<float *>(lds));
    }
  });
}

// ---------------------------------------------------------------------------
// Narrow tiles of up to 16 columns, on the 16 x 16 matrix instructions: half the
// products.  An F32 cache needs that (two contexts of 32k keys, 28 heads on 4:
// 72 us with 32 columns, whose fp32 products take as long as the loads; 55);
// with a BF16 cache it is a microsecond of a 4k-key token.
template <int NK, bool BF>
struct Shape16 {
  static constexpr int KP = BF ? (NK + 1) / 2 : NK;  // 16-byte pieces of a key per quarter-wave
  static constexpr int VP = BF ? 1 : 2;              // pieces of a unit's values per channel and quarter-wave
  static constexpr int QL = BF ? 3 : 1;
  static constexpr int Q_BYTES = QL * KP * 64 * 16;
};
template <int NK, bool BF>
__device__ __forceinline__ void narrow16_body(const Args &g, int me) {
  using S = Shape16<NK, BF>;
  constexpr int dim = NK * 16, row = dim + 4, elem = BF ? 2 : 4, E = BF ? 8 : 4, chunks = dim / E;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ float wave_m[4][16], wave_l[4][16];
  __shared__ uint32_t redo;
  __shared__ Owner slow_owner;
  __shared__ Piece slow_piece;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, quarter = lane >> 4;
  const PagedCache &cache = g.a.c;
  const int run = cache.page_size * dim * elem;
  const size_t page_bytes = size_t(2) * cache.kv_heads * run;
  const uint32_t k_lane = quarter * 256 + col * 16;
  const uint32_t k_tail = BF && NK % 2 && quarter >= 2 ? k_lane - 512 : k_lane;  // an odd NK's last step: q is zero there
  const uint32_t v_lane = cache.kv_heads * run + quarter * dim * 16 + col * 16;
  const u32x4 *qf = reinterpret_cast<const u32x4 *>(lds) + lane;

  for_pieces<kNarrow, kThreads>(g, me, [&](const Owner &w, const Piece &p) {
    const int last = p.unit0 + p.units;
    u32x4 kf[S::KP][2];
    const uint8_t *base = nullptr;
    auto keys = [&] {
#pragma unroll
      for (int i = 0; i < S::KP; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          kf[i][b] = load16(base, (i == S::KP - 1 ? k_tail : k_lane) + i * 1024 + b * 16 * dim * elem);
    };
    if (p.unit0 + wave < last) {
      base = unit_base(g, w, p.h, p.unit0 + wave, run, page_bytes, dim * elem);
      keys();
    }
    __syncthreads();  // LDS is free
    for (int i = tid; i < S::KP * 64; i += kThreads) {
      const int c = i & 15, chunk = i >> 4;
      u32x4 x[S::QL];
      const bool in = c < p.cols && chunk < chunks;
      if (in) load_q<BF>(g, g.a.q + column_place(g, w, p, c), chunk, x);
#pragma unroll
      for (int j = 0; j < S::QL; ++j) reinterpret_cast<u32x4 *>(lds)[j * S::KP * 64 + i] = in ? x[j] : u32x4(0u);
    }
    if (tid == 0) redo = 0;
    int low = 0, high = 0x7fffffff, r;
    if (col < p.cols) column_keys(g, w, col, r, low, high);
    __syncthreads();
    float m = -INFINITY, l = 0.0f;
    f32x4 o[NK];
#pragma unroll
    for (int t = 0; t < NK; ++t) o[t] = f32x4(0.0f);
    for (int u = p.unit0 + wave; u < last; u += 4) {
      u32x4 vf[NK][S::VP];
#pragma unroll
      for (int t = 0; t < NK; ++t)
#pragma unroll
        for (int b = 0; b < S::VP; ++b) vf[t][b] = load16(base, v_lane + t * 256 + b * 16 * dim * elem);
      f32x4 s2[2] = {f32x4(0.0f), f32x4(0.0f)};
      u32x4 qc[S::QL], qn[S::QL];
#pragma unroll
      for (int x = 0; x < S::QL; ++x) qc[x] = qf[x * S::KP * 64];
#pragma unroll
      for (int i = 0; i < S::KP; ++i) {
#pragma unroll
        for (int x = 0; x < S::QL; ++x) qn[x] = qf[(x * S::KP + min(i + 1, S::KP - 1)) * 64];
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BF) {
#pragma unroll
          for (int x = 2; x >= 0; --x)
#pragma unroll
            for (int b = 0; b < 2; ++b) s2[b] = mfma16(kf[i][b], qc[x], s2[b]);
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) s2[b] = mfma16x4(kf[i][b], qc[0], s2[b]);
        }
#pragma unroll
        for (int x = 0; x < S::QL; ++x) qc[x] = qn[x];
      }
      if (u + 4 < last) {
        base = unit_base(g, w, p.h, u + 4, run, page_bytes, dim * elem);
        keys();
      }
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = s2[i >> 2][i & 3];
      soften16<NK>(g, m, l, o, s, u * kUnit, low, high, quarter);
      if (u * kUnit < p.low || (u + 1) * kUnit > p.high)  // what is behind the last key may be anything
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
          for (int b = 0; b < S::VP; ++b) clear_outside<BF>(vf[t][b], u * kUnit, 4 * b + quarter, p.low, p.high);
      u32x4 pw[BF ? 3 : 2];
      weights16<BF>(s, pw);
      if constexpr (BF) {
#pragma unroll
        for (int x = 2; x >= 0; --x)
#pragma unroll
          for (int t = 0; t < NK; ++t) o[t] = mfma16(vf[t][0], pw[x], o[t]);
      } else {
#pragma unroll
        for (int t = 0; t < NK; ++t)
#pragma unroll
          for (int b = 0; b < 2; ++b) o[t] = mfma16x4(vf[t][b], pw[b], o[t]);
      }
    }
    l += dev::xor_lanes<16>(l);
    l += dev::xor_lanes<32>(l);
    if (quarter == 0) wave_m[wave][col] = m;
    __syncthreads();  // q is not needed any more
    const float keep = wave_scale(wave_m, col, m);
    if (quarter == 0) wave_l[wave][col] = l * keep;
    float *os = reinterpret_cast<float *>(lds);
    if (col < p.cols)
#pragma unroll
      for (int t = 0; t < NK; ++t)
        *reinterpret_cast<f32x4 *>(os + (wave * 16 + col) * row + t * 16 + 4 * quarter) = o[t] * keep;
    __syncthreads();
    join_waves<dim>(g, w, p, os, wave_m, wave_l, redo);
    __syncthreads();
    if (const uint32_t again = uniform(int(redo))) {
      slow_owner = w;
      slow_piece = p;
      __syncthreads();
      for (int c = 0; c < p.cols; ++c)
        if (again >> c & 1)
          slow_column<E>((const Args *)__builtin_amdgcn_kernarg_segment_ptr(), &slow_owner, &slow_piece, c,
                            reinterpret_cast<float *>(lds));
    }
  });
}

// ---------------------------------------------------------------------------
// Wide: tiles of 128 columns, 32 per wave, q in registers (of a BF16 cache's
// three planes the lowest in LDS: 256 registers hold two); the units go
// through LDS, one on its way in registers while another is multiplied.
template <int NK, bool BF>
__device__ __forceinline__ void wide_body(const Args &g, int me) {
  using S = Shape<NK, BF>;
  constexpr int dim = NK * 16, ND = S::ND, row = dim + 4, elem = BF ? 2 : 4;
  constexpr int kBytes = kUnit * dim * elem, skew = 128;  // a unit's keys (and values); see below
  constexpr int kLoads = (kBytes / 16 + kThreads - 1) / kThreads;
  constexpr int kStage = 2 * kBytes + skew, kPlane = S::KP * 64;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ uint32_t redo[4];
  __shared__ Owner slow_owner;
  __shared__ Piece slow_piece;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 31, half = lane >> 5;
  const PagedCache &cache = g.a.c;
  const int run = cache.page_size * dim * elem;
  const size_t page_bytes = size_t(2) * cache.kv_heads * run;
  // The second block of 16 keys lies `skew` bytes further on: a quarter-wave
  // reads 8 keys of either, 128 bytes each, and they shall not meet in a bank.
  const int key = tile_key<BF>(col);
  const int k_lane = (key >> 4) * (16 * dim * elem + skew) + (half * 16 + (key & 15)) * 16;
  const int v_lane = kBytes + skew + half * dim * 16 + col * 16;
  const int v_last = NK % 2 && col >= 16 ? v_lane - 256 : v_lane;
  u32x4 *q_lo = reinterpret_cast<u32x4 *>(lds + 2 * kStage) + wave * kPlane + lane;

  for_pieces<kWide, kThreads>(g, me, [&](const Owner &w, const Piece &p) {
    const int c = wave * 32 + col, last = p.unit0 + p.units;
    const bool idle = wave * 32 >= p.cols;
    u32x4 kr[kLoads], vr[kLoads];
    auto request = [&](int u) {
      const uint8_t *kb = unit_base(g, w, p.h, u, run, page_bytes, dim * elem);
      const uint8_t *vb = kb + size_t(cache.kv_heads) * run;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = min((i * kThreads + tid) * 16, kBytes - 16);
        kr[i] = *reinterpret_cast<const u32x4 *>(kb + at);
        vr[i] = *reinterpret_cast<const u32x4 *>(vb + at);
      }
    };
    auto deposit = [&](uint8_t *stage, int u) {
      const bool edge = u * kUnit < p.low || (u + 1) * kUnit > p.high;  // what is behind the last key may be anything
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = (i * kThreads + tid) * 16;
        if (edge) clear_outside<BF>(vr[i], u * kUnit, at / (16 * dim), p.low, p.high);
        if (at < kBytes) {
          *reinterpret_cast<u32x4 *>(stage + at + (at >= kBytes / 2 ? skew : 0)) = kr[i];
          *reinterpret_cast<u32x4 *>(stage + kBytes + skew + at) = vr[i];
        }
      }
    };
    request(p.unit0);
    __syncthreads();  // LDS is free
    if (tid < 4) redo[tid] = 0;
    u32x4 qf[BF ? 2 * S::KP : S::KP];
    int low = 0, high = 0x7fffffff, r;
    if (c < p.cols) column_keys(g, w, p.c0 + c, r, low, high);
    {
      // All of q is requested before any of it is split.
      const float *q = g.a.q + column_place(g, w, p, min(c, p.cols - 1));
      QRaw<BF> raw[S::KP];
#pragma unroll
      for (int i = 0; i < S::KP; ++i) raw[i] = QRaw<BF>(q, 2 * i + half);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < S::KP; ++i) {
        u32x4 x[S::QL];
        raw[i].split(g, x);
        if constexpr (BF) {
          qf[2 * i] = x[0];
          qf[2 * i + 1] = x[1];
          q_lo[i * 64] = x[2];
        } else {
          qf[i] = x[0];
        }
      }
    }
    Running<ND> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t) st.o[t] = f32x16(0.0f);
    deposit(lds, p.unit0);
    if (p.unit0 + 1 < last) request(p.unit0 + 1);
    for (int u = p.unit0; u < last; ++u) {
      __syncthreads();  // this unit is there, the other stage has been read
      const uint8_t *stage = lds + ((u - p.unit0) & 1) * kStage;
      if (u + 1 < last) {
        deposit(lds + ((u - p.unit0 + 1) & 1) * kStage, u + 1);
        if (u + 2 < last) request(u + 2);
      }
      if (idle || !__ballot(c < p.cols && u * kUnit < high && (u + 1) * kUnit > low)) continue;  // nothing to see
      // The next step's operands are on their way from LDS while one is
      // multiplied (left alone, the compiler reads, waits and multiplies).
      f32x16 s(0.0f);
      u32x4 kf = *reinterpret_cast<const u32x4 *>(stage + k_lane), ql{};
      if constexpr (BF) ql = q_lo[0];
#pragma unroll
      for (int i = 0; i < S::KP; ++i) {
        const int next = min(i + 1, S::KP - 1);
        const u32x4 kn = *reinterpret_cast<const u32x4 *>(stage + k_lane + next * 512);
        u32x4 qn{};
        if constexpr (BF) qn = q_lo[next * 64];
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BF) {
          s = mfma(kf, ql, s);
          s = mfma(kf, qf[2 * i + 1], s);
          s = mfma(kf, qf[2 * i], s);
        } else {
          s = mfma4(kf, qf[i], s);
        }
        kf = kn;
        ql = qn;
      }
      u32x4 vf[S::VP], vn[S::VP];
      auto values = [&](int t, u32x4(&v)[S::VP]) {
#pragma unroll
        for (int i = 0; i < S::VP; ++i)
          v[i] = *reinterpret_cast<const u32x4 *>(stage + (t == ND - 1 ? v_last : v_lane) + t * 512 + i * dim * 32);
      };
      values(0, vf);
      soften<BF, ND>(g, st, s, u * kUnit, low, high, half);
      const Weights<BF> pw(s);
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        values(min(t + 1, ND - 1), vn);
        __builtin_amdgcn_sched_barrier(0);
        st.o[t] = pw.times(vf, st.o[t]);
#pragma unroll
        for (int i = 0; i < S::VP; ++i) vf[i] = vn[i];
      }
    }
    st.l += dev::xor_lanes<32>(st.l);
    bool nan = st.l != st.l;
    const float inv = st.l > 0.0f ? 1.0f / st.l : 0.0f;
    if (c < p.cols) {
      float *part = p.part ? p.part + size_t(c) * row : g.a.out + column_place(g, w, p, c);
      if (p.part && half == 0) {
        part[dim] = st.m;
        part[dim + 1] = st.l;
      }
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int d = t * 32 + 8 * a + 4 * half;
          if (d < dim) {
            f32x4 x = {st.o[t][4 * a], st.o[t][4 * a + 1], st.o[t][4 * a + 2], st.o[t][4 * a + 3]};
            nan |= x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
            if (!p.part) x *= inv;
            *reinterpret_cast<f32x4 *>(part + d) = x;
          }
        }
      if (nan) atomicOr(&redo[wave], 1u << col);
    }
    __syncthreads();
    for (int x = 0; x < 4; ++x)
      if (const uint32_t again = uniform(int(redo[x]))) {
        slow_owner = w;
        slow_piece = p;
        __syncthreads();
        for (int y = 0; y < 32; ++y)
          if (again >> y & 1)
            slow_column<S::E>((const Args *)__builtin_amdgcn_kernarg_segment_ptr(), &slow_owner, &slow_piece, x * 32 + y,
                              reinterpret_cast<float *>(lds));
      }
  });
}

// ---------------------------------------------------------------------------
template <int NK, bool BF>
__global__ __launch_bounds__(kThreads, NK <= (BF ? 8 : 5) ? 2 : 1) void k_paged_narrow(const Args g) {
  narrow_body<NK, BF>(g, blockIdx.x);
}
template <int NK, bool BF>
__global__ __launch_bounds__(kThreads, (NK <= (BF ? 6 : 4) ? 3 : NK <= 8 ? 2 : 1)) void k_paged_narrow16(const Args g) {
  narrow16_body<NK, BF>(g, blockIdx.x);
}
// Both kinds of tiles in one launch, the wide ones first: the narrow ones fill
// what they leave.  (Two launches, of which one may find nothing to do: 5 us.)
template <int NK, bool BF, bool N16>
__global__ __launch_bounds__(kThreads, (BF || N16 || NK <= 5 ? 2 : 1)) void k_paged_both(const Args g) {
  const int me = blockIdx.x;
  if (me < g.workers) wide_body<NK, BF>(g, me);
  else if constexpr (N16) narrow16_body<NK, BF>(g, me - g.workers);
  else narrow_body<NK, BF>(g, me - g.workers);
}

// ---------------------------------------------------------------------------
// Wide heads (more than 128 channels): the same with 16 columns per wave, eight
// waves, on the 16 x 16 matrix instructions.  32 columns' output and q would
// take all registers of a wave with a SIMD to itself, and nothing would run
// beside its waits; two waves of 16 columns share a SIMD.
constexpr int kThreads16 = 512;
template <int NK, bool BF>
__global__ __launch_bounds__(kThreads16, 2) void k_paged_wide16(const Args g) {
  const int me = blockIdx.x;
  constexpr int dim = NK * 16, row = dim + 4, elem = BF ? 2 : 4, E = BF ? 8 : 4;
  constexpr int KP = BF ? (NK + 1) / 2 : NK;  // 16-byte pieces of a key per quarter-wave
  constexpr int chunks = dim / E;
  constexpr int kBytes = kUnit * dim * elem, kStage = 2 * kBytes;
  constexpr int kLoads = (kBytes / 16 + kThreads16 - 1) / kThreads16;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ uint32_t redo[8];
  __shared__ Owner slow_owner;
  __shared__ Piece slow_piece;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), col = lane & 15, quarter = lane >> 4;
  const PagedCache &cache = g.a.c;
  const int run = cache.page_size * dim * elem;
  const size_t page_bytes = size_t(2) * cache.kv_heads * run;
  const int k_lane = quarter * 256 + col * 16;
  const int v_lane = kBytes + quarter * dim * 16 + col * 16;

  for_pieces<kWide, kThreads16>(g, me, [&](const Owner &w, const Piece &p) {
    const int c = wave * 16 + col, last = p.unit0 + p.units;
    const bool idle = wave * 16 >= p.cols;
    u32x4 kr[kLoads], vr[kLoads];
    auto request = [&](int u) {
      const uint8_t *kb = unit_base(g, w, p.h, u, run, page_bytes, dim * elem);
      const uint8_t *vb = kb + size_t(cache.kv_heads) * run;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = min((i * kThreads16 + tid) * 16, kBytes - 16);
        kr[i] = *reinterpret_cast<const u32x4 *>(kb + at);
        vr[i] = *reinterpret_cast<const u32x4 *>(vb + at);
      }
    };
    auto deposit = [&](uint8_t *stage, int u) {
      const bool edge = u * kUnit < p.low || (u + 1) * kUnit > p.high;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = (i * kThreads16 + tid) * 16;
        if (edge) clear_outside<BF>(vr[i], u * kUnit, at / (16 * dim), p.low, p.high);
        if (at < kBytes) {
          *reinterpret_cast<u32x4 *>(stage + at) = kr[i];
          *reinterpret_cast<u32x4 *>(stage + kBytes + at) = vr[i];
        }
      }
    };
    request(p.unit0);
    __syncthreads();  // LDS is free
    if (tid < 8) redo[tid] = 0;
    u32x4 qf[KP][BF ? 3 : 1];
    int low = 0, high = 0x7fffffff, r;
    if (c < p.cols) column_keys(g, w, p.c0 + c, r, low, high);
    {
      const float *q = g.a.q + column_place(g, w, p, min(c, p.cols - 1));
      QRaw<BF> raw[KP];
#pragma unroll
      for (int i = 0; i < KP; ++i) raw[i] = QRaw<BF>(q, min(4 * i + quarter, chunks - 1));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        raw[i].split(g, qf[i]);  // an odd NK's last step has two pieces: zeros times any
        if (BF && NK % 2 && i == KP - 1 && quarter >= 2)
#pragma unroll
          for (int x = 0; x < (BF ? 3 : 1); ++x) qf[i][x] = u32x4(0u);
      }
    }
    const int k_tail = BF && NK % 2 && quarter >= 2 ? k_lane - 512 : k_lane;
    float m = -INFINITY, l = 0.0f;
    f32x4 o[NK];
#pragma unroll
    for (int t = 0; t < NK; ++t) o[t] = f32x4(0.0f);
    deposit(lds, p.unit0);
    if (p.unit0 + 1 < last) request(p.unit0 + 1);
    for (int u = p.unit0; u < last; ++u) {
      __syncthreads();  // this unit is there, the other stage has been read
      const uint8_t *stage = lds + ((u - p.unit0) & 1) * kStage;
      if (u + 1 < last) {
        deposit(lds + ((u - p.unit0 + 1) & 1) * kStage, u + 1);
        if (u + 2 < last) request(u + 2);
      }
      const int base = u * kUnit;
      if (idle || !__ballot(c < p.cols && base < high && base + kUnit > low)) continue;  // nothing to see
      f32x4 s2[2] = {f32x4(0.0f), f32x4(0.0f)};
      auto keys = [&](int i, u32x4(&k)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
          k[b] = *reinterpret_cast<const u32x4 *>(stage + b * (kBytes / 2) + (i == KP - 1 ? k_tail : k_lane) + i * 1024);
      };
      u32x4 kf[2], kn[2];
      keys(0, kf);
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        keys(min(i + 1, KP - 1), kn);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BF) {
#pragma unroll
          for (int x = 2; x >= 0; --x)
#pragma unroll
            for (int b = 0; b < 2; ++b) s2[b] = mfma16(kf[b], qf[i][x], s2[b]);
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) s2[b] = mfma16x4(kf[b], qf[i][0], s2[b]);
        }
        kf[0] = kn[0];
        kf[1] = kn[1];
      }
      constexpr int VP = BF ? 1 : 2;
      auto values = [&](int t, u32x4(&v)[2 * VP]) {  // of two channel tiles
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int b = 0; b < VP; ++b)
            v[x * VP + b] = *reinterpret_cast<const u32x4 *>(stage + v_lane + b * (kBytes / 2) + min(t + x, NK - 1) * 256);
      };
      u32x4 vf[2 * VP], vn[2 * VP];
      values(0, vf);
      float s[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = s2[i >> 2][i & 3];
      soften16<NK>(g, m, l, o, s, base, low, high, quarter);
      u32x4 pw[BF ? 3 : 2];
      weights16<BF>(s, pw);
#pragma unroll
      for (int t = 0; t < NK; t += 2) {
        values(min(t + 2, NK - 1), vn);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (BF) {
#pragma unroll
          for (int x = 2; x >= 0; --x)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (t + y < NK) o[t + y] = mfma16(vf[y], pw[x], o[t + y]);
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (t + y < NK) o[t + y] = mfma16x4(vf[2 * y + b], pw[b], o[t + y]);
        }
#pragma unroll
        for (int i = 0; i < 2 * VP; ++i) vf[i] = vn[i];
      }
    }
    l += dev::xor_lanes<16>(l);
    l += dev::xor_lanes<32>(l);
    bool nan = l != l;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (c < p.cols) {
      float *part = p.part ? p.part + size_t(c) * row : g.a.out + column_place(g, w, p, c);
      if (p.part && quarter == 0) {
        part[dim] = m;
        part[dim + 1] = l;
      }
#pragma unroll
      for (int t = 0; t < NK; ++t) {
        f32x4 x = o[t];
        nan |= x[0] != x[0] || x[1] != x[1] || x[2] != x[2] || x[3] != x[3];
        if (!p.part) x *= inv;
        *reinterpret_cast<f32x4 *>(part + t * 16 + 4 * quarter) = x;
      }
      if (nan) atomicOr(&redo[wave], 1u << col);
    }
    __syncthreads();
    for (int x = 0; x < 8; ++x)
      if (const uint32_t again = uniform(int(redo[x]))) {
        slow_owner = w;
        slow_piece = p;
        __syncthreads();
        for (int y = 0; y < 16; ++y)
          if (again >> y & 1)
            slow_column<E>((const Args *)__builtin_amdgcn_kernarg_segment_ptr(), &slow_owner, &slow_piece, x * 16 + y,
                           reinterpret_cast<float *>(lds));
      }
  });
}

// ---------------------------------------------------------------------------
// Host side.
struct Plan {
  bool narrow, wide;
  int64_t bytes;
  Args g;
};

Plan plan_of(const PagedAttn &a, uint8_t *ws) {
  Plan p;
  const PagedBatch &b = a.b;
  Args &g = p.g;
  g.a = a;
  g.group = a.heads / a.c.kv_heads;
  const int groups = b.prefix_tables ? b.sequences / b.share : 0;
  g.owners = b.sequences + groups;
  const float mul = a.scale > 0.0f ? a.scale : 1.0f / std::sqrt(float(a.c.dim));
  g.qmul = a.softcap > 0.0f ? mul / a.softcap : mul * kLog2e;
  g.smul = a.softcap * kLog2e;
  // Narrow tiles of 16 columns if a row's heads fit, unless many owners (the
  // average sequence, or the groups) would have 17 to 32.
  auto between = [](int64_t cols) { return cols > 16 && cols <= kNarrow; };
  g.narrow = g.group <= 16 && !between(int64_t(b.rows) * g.group / b.sequences) &&
                     !(groups && between(int64_t(b.rows) * g.group / groups))
                 ? 16
                 : kNarrow;
  // Row starts are on the device; without them every sequence has one row.
  p.narrow = b.starts || g.group <= g.narrow;
  p.wide = b.starts ? int64_t(b.rows) * g.group > g.narrow
                    : g.group > g.narrow || (groups && int64_t(b.share) * g.group > g.narrow);
  g.workers = a.c.dim <= 128 ? 512 : 256;
  const int64_t blocks = int64_t(b.rows) * g.group / kWide;
  g.prefix_tiles = int(blocks + b.sequences);
  // Units are counted in 32 bits; the costs and padding that are added leave them below 2^31.
  const int64_t own_units = (int64_t(b.table_pages) * a.c.page_size) / kUnit + 1 + kItemCost<kNarrow>,
                prefix_units = (int64_t(b.prefix_pages) * a.c.page_size) / kUnit + 1 + kItemCost<kNarrow>;
  if (a.c.kv_heads * ((b.sequences + blocks) * own_units + (groups ? (groups + blocks) * prefix_units : 0)) >= kLineMax)
    fail(QNN_E_RANGE, "paged attention: more rows times pages than one call counts");
  const int64_t tiles[2] = {p.narrow ? g.owners : 0, p.wide ? blocks + b.sequences + (groups ? blocks + groups : 0) : 0};
  g.cols[0] = !b.starts && !groups ? std::min(g.group, g.narrow) : g.narrow;
  g.cols[1] = kWide;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    uint8_t *from = ws ? ws + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  for (int c = 0; c < 2; ++c) {
    const int64_t slots = tiles[c] ? 2 * int64_t(g.workers) : 0;
    g.head[c] = reinterpret_cast<Line *>(take(sizeof(Line)));
    g.table[c] = reinterpret_cast<int *>(take(groups ? tiles[c] * 4 : 0));
    g.splits[c] = reinterpret_cast<Split *>(take(tiles[c] ? g.workers * sizeof(Split) : 0));
    g.parts[c] = reinterpret_cast<float *>(take(slots * g.cols[c] * (a.c.dim + 4) * 4));
  }
  g.whole = reinterpret_cast<float *>(take(groups ? int64_t(2) * b.rows * a.heads * (a.c.dim + 4) * 4 : 0));
  g.first_keys = reinterpret_cast<int *>(take(groups && a.window > 0 ? groups * 4 : 0));
  p.bytes = at;
  return p;
}

template <typename K>
void run(K kernel, const Args &g, int workgroups, size_t lds, hipStream_t s, int threads = kThreads) {
  if (lds > 65536)
    hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                  int(lds)),
              "paged attention LDS size");
  kernel<<<workgroups, threads, lds, s>>>(g);
  hip_check(hipGetLastError(), "paged attention launch");
}

template <int NK, bool BF>
void launch(const Plan &p, hipStream_t s) {
  constexpr size_t unit = size_t(kUnit) * NK * 16 * (BF ? 2 : 4);
  constexpr size_t lds16 = std::max<size_t>(Shape16<NK, BF>::Q_BYTES, 4 * 16 * (NK * 16 + 4) * 4),
                   lds32 = std::max<size_t>(Shape<NK, BF>::Q_BYTES, 4 * 32 * (NK * 16 + 4) * 4);
  const bool n16 = p.g.narrow == 16;
  const int workers = p.g.workers;
  if constexpr (NK <= 8) {
    constexpr size_t wide = 2 * (2 * unit + 128) + (BF ? 4 * Shape<NK, BF>::KP * 64 * 16 : 0);
    if (p.wide) {
      if (n16) run(k_paged_both<NK, BF, true>, p.g, p.narrow ? 2 * workers : workers, std::max(wide, lds16), s);
      else run(k_paged_both<NK, BF, false>, p.g, p.narrow ? 2 * workers : workers, std::max(wide, lds32), s);
      return;
    }
  }
  if (p.narrow) {
    if (n16) run(k_paged_narrow16<NK, BF>, p.g, workers, lds16, s);
    else run(k_paged_narrow<NK, BF>, p.g, workers, lds32, s);
  }
  if constexpr (NK > 8)
    if (p.wide) run(k_paged_wide16<NK, BF>, p.g, workers, 4 * unit, s, kThreads16);
}

// The main kernels of a call; the parts are joined by the caller.
template <bool BF>
void launch_main(const Plan &p, hipStream_t s) {
  switch (p.g.a.c.dim / 16) {
#define QNN_PAGED(N) case N: launch<N, BF>(p, s); break;
    QNN_PAGED(1) QNN_PAGED(2) QNN_PAGED(3) QNN_PAGED(4) QNN_PAGED(5) QNN_PAGED(6) QNN_PAGED(7) QNN_PAGED(8)
    QNN_PAGED(9) QNN_PAGED(10) QNN_PAGED(11) QNN_PAGED(12) QNN_PAGED(13) QNN_PAGED(14) QNN_PAGED(15) QNN_PAGED(16)
#undef QNN_PAGED
  }
}

}  // namespace
}  // namespace qnn
