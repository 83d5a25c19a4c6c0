// qnn_paged_attention.hip -- paged attention: BF16 caches, the joining of parts
// and the entry (kernels in qnn_paged_attention_dev.h).
#include "qnn_paged_attention_dev.h"

namespace qnn {
namespace {

// ---------------------------------------------------------------------------
// With prefixes and a window: the first prefix key that any row of a group
// sees, from the row that lies furthest in front.  A launch of its own: every
// workgroup of the others asks for it several times, and a loop over the group
// in each made it 4.5 ms where 1000 sequences share a prefix (0.29 now), 57 us
// at 48 (34); 25.8 us at 8 groups of 4 (27.5).
__global__ __launch_bounds__(kThreads) void k_paged_first_keys(const Args g) {
  __shared__ unsigned most[kThreads / 64];
  const PagedBatch &b = g.a.b;
  const int p = blockIdx.x, tid = threadIdx.x;
  constexpr unsigned kNoRow = 0x3fffffff;  // the largest own position
  unsigned before = 0;                     // the largest distance of a row in front of that
  for (int s = p * b.share + tid; s < (p + 1) * b.share; s += kThreads) {
    int first, end;
    dev::row_range<false>(b, s, first, end);
    if (end > first) before = max(before, kNoRow - unsigned(dev::own_length<false>(b, s) - (end - first)));
  }
  before = dev::wave_max_u32(before);
  if ((tid & 63) == 0) most[tid >> 6] = before;
  __syncthreads();
  if (tid) return;
  for (int x = 1; x < kThreads / 64; ++x) before = max(before, most[x]);
  const int64_t low = int64_t(dev::prefix_length<false>(b, p)) + int(kNoRow - before) - g.a.window + 1;
  g.first_keys[p] = int(max(low, int64_t(0)));
}

// ---------------------------------------------------------------------------
// Joins a column's parts: out = sum of 2^(m - M) o over sum of 2^(m - M) l, M
// the largest m.  WAVES waves share the parts of a column: every wave takes the
// maximum and the sum of all of them (a part per lane), then a lane takes four
// channels of every few parts; what the lane groups have meets in LDS, in order.
struct Parts {
  const float *first, *rest;  // of the column: the first part, the second
  int64_t step;               // to the next
  int n;
};
__device__ __forceinline__ const float *part_at(const Parts &p, int x) {
  return x == 0 ? p.first : p.rest + (x - 1) * p.step;
}
template <int WAVES, int N>
__device__ __forceinline__ void join_column(const Parts (&parts)[N], int dim, float *out, f32x4 *lds) {
  const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6, d4 = dim / 4, groups = 64 / d4;
  const int group = lane / d4, d = lane - group * d4, k = wave * groups + group, step = WAVES * groups;
  const bool mine = group < groups;
  // A part's maximum and sum and the first outputs are all requested at once.
  constexpr int kAhead = 4;
  f32x4 ahead[N][kAhead];
  float ahead_m[N][kAhead];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (mine && k + j * step < parts[i].n) {
        const float *p = part_at(parts[i], k + j * step);
        ahead[i][j] = reinterpret_cast<const f32x4 *>(p)[d];
        ahead_m[i][j] = p[dim];
      }
  float top = -INFINITY, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    for (int x = lane; x < parts[i].n; x += 64) {
      const float *p = part_at(parts[i], x);
      const float m = p[dim], l = p[dim + 1], t = fmaxf(top, m), t0 = t == -INFINITY ? 0.0f : t;
      sum = sum * exp2f(top - t0) + l * exp2f(m - t0);
      top = t;
    }
  const float own = top;
  top = dev::wave_max_xor(top);
  if (top == -INFINITY) top = 0.0f;  // nothing seen, or NaN alone
  sum = dev::wave_sum_xor(own == -INFINITY && sum == 0.0f ? 0.0f : sum * exp2f((own == -INFINITY ? 0.0f : own) - top));
  f32x4 o = f32x4(0.0f);
  if (mine)
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (k + j * step < parts[i].n) o += exp2f(ahead_m[i][j] - top) * ahead[i][j];
      for (int x = k + kAhead * step; x < parts[i].n; x += step) {
        const float *p = part_at(parts[i], x);
        o += exp2f(p[dim] - top) * reinterpret_cast<const f32x4 *>(p)[d];
      }
    }
  lds[wave * 64 + lane] = o;
  if (WAVES > 1) __syncthreads();
  else dev::wave_lds_sync();
  if (wave == 0 && lane < d4) {
    f32x4 all = f32x4(0.0f);
    for (int x = 0; x < WAVES; ++x)
      for (int y = 0; y < groups; ++y) all += lds[x * 64 + y * d4 + lane];
    reinterpret_cast<f32x4 *>(out)[lane] = sum > 0.0f || sum != sum ? all / sum : f32x4(0.0f);
  }
  if (WAVES > 1) __syncthreads();
  else dev::wave_lds_sync();
}

// Without prefixes: the items that are split, a worker's per blockIdx.x.
// Narrow ones have many parts and few columns: a workgroup per column.
__device__ __forceinline__ size_t split_place(const Args &g, const Split &s, int c) {
  Owner w;
  w.first = s.first;
  Piece p;
  p.h = s.h;
  p.c0 = s.c0;
  return column_place(g, w, p, c);
}
__device__ __forceinline__ void join_narrow(const Args &g, int from, int y, int ys) {
  __shared__ f32x4 lds[kThreads];
  const int dim = g.a.c.dim;
  const Split s = g.splits[0][from];
  const int n = min(s.n, g.workers - from);
  if (n <= 0) return;
  for (int c = y; c < s.cols; c += ys) {
    const int64_t slot = int64_t(g.cols[0]) * (dim + 4);
    const float *at = g.parts[0] + (2 * int64_t(from) + 1) * slot + size_t(c) * (dim + 4);
    const Parts parts[1] = {{at, at + slot, 2 * slot, n}};
    join_column<4>(parts, dim, g.a.out + split_place(g, s, c), lds);
  }
}
// Wide ones have few parts and many columns: a thread per column and four
// channels, four parts on their way at once.  (With a wave per column, 33 us
// for 256 items of two parts.)
__device__ __forceinline__ void join_wide(const Args &g, int from, int y, int ys) {
  const int dim = g.a.c.dim, d4 = dim / 4;
  const Split s = g.splits[1][from];
  const int n = min(s.n, g.workers - from);
  if (n <= 0) return;
  const int64_t slot = int64_t(g.cols[1]) * (dim + 4);
  for (int i = y * kThreads + threadIdx.x; i < s.cols * d4; i += ys * kThreads) {
    const int c = i / d4, d = i - c * d4;
    const float *at = g.parts[1] + (2 * int64_t(from) + 1) * slot + size_t(c) * (dim + 4);
    float top = -INFINITY, l = 0.0f;
    f32x4 o = f32x4(0.0f);
    for (int x0 = 0; x0 < n; x0 += 4) {
      float m[4], ls[4];
      f32x4 os[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int y = min(x0 + x, n - 1);  // a part again where there are no more: its weight is zero
        const float *p = y == 0 ? at : at + (2 * y - 1) * slot;
        m[x] = p[dim];
        ls[x] = p[dim + 1];
        os[x] = reinterpret_cast<const f32x4 *>(p)[d];
      }
      const float old = top;
#pragma unroll
      for (int x = 0; x < 4; ++x) top = fmaxf(top, m[x]);
      const float t0 = top == -INFINITY ? 0.0f : top, keep = exp2f(old - t0);
      l *= keep;
      o *= keep;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (x0 + x < n) {
          const float e = exp2f(m[x] - t0);
          l += e * ls[x];
          o += e * os[x];
        }
    }
    reinterpret_cast<f32x4 *>(g.a.out + split_place(g, s, c))[d] = l > 0.0f || l != l ? o / l : f32x4(0.0f);
  }
}

// Rows of the grid: `narrow` for the narrow tiles, the others for the wide ones.
__global__ __launch_bounds__(kThreads) void k_paged_join_splits(const Args g, int narrow) {
  const int y = blockIdx.y;
  if (y < narrow) join_narrow(g, blockIdx.x, y, narrow);
  else join_wide(g, blockIdx.x, y - narrow, gridDim.y - narrow);
}

// With prefixes: every row and head.  The parts of a column's item: none if it
// has no keys; false if its one part is the result already.
template <int C>
__device__ __forceinline__ bool parts_of(const Args &g, const Owner &w, int o, int c, int h, Parts &p) {
  constexpr int CT = C ? kWide : kNarrow;
  const int tile = c / CT, units = tile_units<CT>(g, w, tile);
  p.n = 0;
  if (units == 0) return true;
  const int id = first_tile_id<CT>(g, w, o) + tile;
  const Line line = *g.head[C];
  const unsigned share = max(line.share, 1), at = unsigned(max(g.table[C][id] + h * padded<CT>(line, units), 0));
  const int last = g.workers - 1, w0 = min(int(at / share), last);
  const int64_t slot = int64_t(g.cols[C]) * (g.a.c.dim + 4);
  p.n = min(int((at + units - 1) / share), last) - w0 + 1;
  p.first = p.n == 1 ? whole_part(g, w.prefix_group >= 0, h, int64_t(w.first) * g.group + c)
                     : split_part(g, C, w0, false) + size_t(c % CT) * (g.a.c.dim + 4);
  p.rest = p.first + slot;  // the next worker's first slot
  p.step = 2 * slot;
  return p.n > 1 || w.prefix > 0;
}

__global__ __launch_bounds__(kThreads) void k_paged_join(const Args g) {
  __shared__ f32x4 lds[kThreads];
  const PagedBatch &b = g.a.b;
  const int row = blockIdx.x, head = blockIdx.y, h = head / g.group;
  const int s = uniform(row_sequence(b, row)), prefix = b.sequences + s / b.share;
  const Owner own = owner_of(g, s), w = owner_of(g, prefix);
  if (row < own.first || row >= own.end) return;
  Parts parts[2];
  const int c = (row - own.first) * g.group + head % g.group, pc = (row - w.first) * g.group + head % g.group;
  if (!(own.cols > g.narrow ? parts_of<1>(g, own, s, c, h, parts[0]) : parts_of<0>(g, own, s, c, h, parts[0]))) return;
  parts[1].n = 0;
  if (row < w.first || row >= w.end) {  // row starts that do not ascend (reported where they were read)
  } else if (w.cols > g.narrow) {
    parts_of<1>(g, w, prefix, pc, h, parts[1]);
  } else {
    parts_of<0>(g, w, prefix, pc, h, parts[1]);
  }
  join_column<4>(parts, g.a.c.dim, g.a.out + (size_t(row) * g.a.heads + head) * g.a.c.dim, lds);
}

}  // namespace

size_t paged_attention_bytes(const PagedAttn &a) { return size_t(plan_of(a, nullptr).bytes); }

void paged_attention_launch(const PagedAttn &a, void *ws, hipStream_t s) {
  const Plan p = plan_of(a, static_cast<uint8_t *>(ws));
  if (a.b.prefix_tables && a.window > 0) {
    k_paged_first_keys<<<a.b.sequences / a.b.share, kThreads, 0, s>>>(p.g);
    hip_check(hipGetLastError(), "paged attention window launch");
  }
  if (a.c.bf16) launch_main<true>(p, s);
  else paged_attention_f32_launch(a, ws, s);
  if (a.b.prefix_tables) {
    k_paged_join<<<dim3(a.b.rows, a.heads), kThreads, 0, s>>>(p.g);
  } else {
    const int narrow = p.narrow ? std::min(p.g.cols[0], 8) : 0,
              wide = p.wide ? std::max(1, a.c.dim * kWide / 4 / kThreads) : 0;
    k_paged_join_splits<<<dim3(p.g.workers, narrow + wide), kThreads, 0, s>>>(p.g, narrow);
  }
  hip_check(hipGetLastError(), "paged attention join launch");
}

}  // namespace qnn
