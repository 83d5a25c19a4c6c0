// qnn_paged.hip -- the paged KV cache of several sequences: append with RoPE,
// advancing lengths, and following a beam search's parents.
//
// Row i of sequence s (n rows, `length` own keys including them, P keys of its
// group's shared prefix) has own position length - n + i, kept in the
// sequence's pages, and absolute position P + length - n + i, which the
// rotation takes.
#include <cmath>

#include "qnn_paged_dev.h"

namespace qnn {
namespace {

// ---------------------------------------------------------------------------
// Append: q and k rotated by their absolute position, k and v written to the
// pages.  The rotation is k_rope's (qnn_decode.hip): angle, sine, cosine and
// products in double, rounded once; a BF16 cache rounds that fp32 value (and
// v) to nearest even, half a step of 2^-8, as the storage type demands.
constexpr int kAppendThreads = 256;
constexpr int kAppendMaxDim = 256;

// The sequence of a row, or -1 for rows behind the last sequence.
__device__ __forceinline__ int row_sequence(const PagedBatch &b, int row) {
  if (!b.starts) return row;
  int lo = 0, hi = b.sequences;  // starts[lo] <= row < starts[hi], where they ascend
  if (row < b.starts[0] || row >= b.starts[hi]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (b.starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The searches for a row's or group's sequence meet only some sequences where
// row starts do not ascend, and none without rows: with row starts, the last
// workgroups of a launch look at every sequence's data, a thread each, and do
// nothing else.  (In the others, it was 1 us of 41.)
__host__ __device__ __forceinline__ int report_groups(const PagedBatch &b) {
  return b.starts ? (b.sequences + kAppendThreads - 1) / kAppendThreads : 0;
}
__device__ __forceinline__ bool report_batch(const PagedBatch &b) {
  const int group = int(blockIdx.x) - int(gridDim.x) + report_groups(b), s = group * kAppendThreads + threadIdx.x;
  if (group < 0) return false;
  if (blockIdx.y == 0 && s < b.sequences) {
    int first, end;
    dev::row_range(b, s, first, end);
    dev::own_length(b, s);
    dev::prefix_length(b, s / b.share);
  }
  return true;
}

template <int E, typename T>
__global__ __launch_bounds__(kAppendThreads) void k_paged_append(const PagedCache c, const PagedBatch b, const float *k,
                                                                 const float *v, const float *q, float *q_out, int heads,
                                                                 float theta) {
#pragma clang fp contract(off)
  __shared__ double cs[kAppendMaxDim / 2], sn[kAppendMaxDim / 2];
  const int row = blockIdx.x, dim = c.dim, half = dim / 2, tid = threadIdx.x;
  if (report_batch(b)) return;
  const int s = row_sequence(b, row);
  if (s < 0) return;
  int first, end;
  dev::row_range(b, s, first, end);
  if (row < first || row >= end) return;  // starts that do not ascend
  const int own = dev::own_length(b, s) - end + row, at = own + dev::prefix_length(b, s / b.share);
  if (own < 0) {  // more rows than keys
    if (tid == 0) atomicOr(b.err, kPagedErr);
    return;
  }
  const bool turn = theta > 0.0f;
  if (turn)
    for (int j = tid; j < half; j += kAppendThreads) {
      const double angle = double(at) * pow(double(theta), -2.0 * double(j) / double(dim));
      double sv, cv;
      sincos(angle, &sv, &cv);
      cs[j] = cv;
      sn[j] = sv;
    }
  __syncthreads();
  auto rotate = [&](const float *src, int j, float &x, float &y) {
    const float a = src[j], e = src[j + half];
    if (!turn) {
      x = a;
      y = e;
      return;
    }
    x = float(double(a) * cs[j] - double(e) * sn[j]);
    y = float(double(a) * sn[j] + double(e) * cs[j]);
  };
  const int work = blockIdx.y * kAppendThreads + tid, stride = gridDim.y * kAppendThreads;
  if (q)
    for (int i = work; i < heads * half; i += stride) {
      const size_t at_q = (size_t(row) * heads + i / half) * dim;
      float x, y;
      rotate(q + at_q, i % half, x, y);
      q_out[at_q + i % half] = x;
      q_out[at_q + i % half + half] = y;
    }
  const int page = dev::checked_page(b.tables[size_t(s) * b.table_pages + (own >> b.page_shift)], b);
  if (page < 0) return;
  const int t = own & (c.page_size - 1), head = c.page_size * dim;
  T *base = static_cast<T *>(c.pages) + size_t(page) * 2 * c.kv_heads * head;
  for (int i = work; i < c.kv_heads * half; i += stride) {
    const int h = i / half, j = i % half;
    float x, y;
    rotate(k + (size_t(row) * c.kv_heads + h) * dim, j, x, y);
    base[h * head + dev::key_place<E>(t, j, dim)] = T(x);
    base[h * head + dev::key_place<E>(t, j + half, dim)] = T(y);
  }
  for (int i = work; i < c.kv_heads * dim; i += stride)
    base[(c.kv_heads + i / dim) * head + dev::value_place<E>(t, i % dim, dim)] =
        T(v[size_t(row) * c.kv_heads * dim + i]);
}

// Many rows: a workgroup takes the tokens of a call that lie in one group of 32
// own positions of a sequence, so that values are written in whole pieces of 8
// (4) tokens, and a part of their heads.  Sines and cosines of a channel pair
// come from one power and two sincos per thread, then e^(i (t + 1) f) =
// e^(i t f) e^(i f) in double over its tokens (at most 16 steps of 2^-53 each,
// far below the fp32 rounding).
// A sequence's groups have the ids from first row / 32 + 2 s on.
constexpr int kAppendGroup = 32;
__device__ __forceinline__ int first_group(const PagedBatch &b, int s) {
  return dev::first_row(b, s) / kAppendGroup + 2 * s;
}

template <int E, typename T>
__global__ __launch_bounds__(kAppendThreads) void k_paged_append_groups(const PagedCache c, const PagedBatch b,
                                                                        const float *k, const float *v, const float *q,
                                                                        float *q_out, int heads, float theta) {
#pragma clang fp contract(off)
  extern __shared__ double2 turn[];  // [32 tokens][dim / 2]
  const int id = blockIdx.x, dim = c.dim, half = dim / 2, tid = threadIdx.x;
  if (report_batch(b)) return;
  int s = 0;
  for (int step = 1 << 16; step; step >>= 1)  // the last sequence whose first group is not behind this one
    if (s + step < b.sequences && first_group(b, s + step) <= id) s += step;
  int first, end;
  dev::row_range<false>(b, s, first, end);
  const int length = dev::own_length<false>(b, s), start = length - (end - first);  // own position of row `first`
  if (first == end) return;
  if (start < 0) {  // more rows than keys
    if (tid == 0) atomicOr(b.err, kPagedErr);
    return;
  }
  const int base = (start / kAppendGroup + id - first_group(b, s)) * kAppendGroup;  // first position of the group
  const int low = max(base, start), high = min(base + kAppendGroup, length);
  if (low >= high) return;
  const int row0 = first + low - start, count = high - low;  // rows row0 .. row0 + count - 1 at positions low ..
  if (theta > 0.0f) {
    const int parts = min(kAppendThreads / half, kAppendGroup), per = (kAppendGroup + parts - 1) / parts;
    const int j = tid % half, part = tid / half;
    if (part < parts) {
      const double f = pow(double(theta), -2.0 * double(j) / double(dim));
      const int t0 = part * per;
      double sn, cn, ss, cs;
      sincos(double(low + t0 + dev::prefix_length<false>(b, s / b.share)) * f, &sn, &cn);
      sincos(f, &ss, &cs);
      for (int t = t0; t < min(t0 + per, count); ++t) {
        turn[t * half + j] = {cn, sn};
        const double c1 = cn * cs - sn * ss;
        sn = sn * cs + cn * ss;
        cn = c1;
      }
    }
    __syncthreads();
  }
  const int page = dev::checked_page(b.tables[size_t(s) * b.table_pages + (base >> b.page_shift)], b);
  const int head = c.page_size * dim, t_low = low & (c.page_size - 1);
  T *pages = static_cast<T *>(c.pages) + size_t(max(page, 0)) * 2 * c.kv_heads * head;
  const int work = blockIdx.y * kAppendThreads + tid, stride = gridDim.y * kAppendThreads;
  // N channels from d and their partners of a token and head, rotated.
  auto load = [&](const float *src, int t, int d, auto &lo, auto &hi) {
    constexpr int N = sizeof(lo) / 4;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      *reinterpret_cast<float4 *>(lo + e) = *reinterpret_cast<const float4 *>(src + d + e);
      *reinterpret_cast<float4 *>(hi + e) = *reinterpret_cast<const float4 *>(src + d + half + e);
    }
    if (theta > 0.0f)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double2 z = turn[t * half + d + e];
        const double x = lo[e], y = hi[e];
        lo[e] = float(x * z.x - y * z.y);
        hi[e] = float(x * z.y + y * z.x);
      }
  };
  // q: four channels per thread, rows read and written in runs.
  if (q) {
    const int chunks = half / 4, n = count * heads * chunks;
#pragma unroll 2
    for (int i = work; i < n; i += stride) {
      const int d = i % chunks * 4, y = i / chunks, t = y / heads;
      const size_t at = (size_t(row0) * heads + y) * dim;
      alignas(16) float lo[4], hi[4];
      load(q + at, t, d, lo, hi);
      *reinterpret_cast<float4 *>(q_out + at + d) = *reinterpret_cast<const float4 *>(lo);
      *reinterpret_cast<float4 *>(q_out + at + d + half) = *reinterpret_cast<const float4 *>(hi);
    }
  }
  if (page < 0) return;
  // k: a wave has 16 tokens by a few chunks of E channels: runs of 16 pieces to
  // write, whole lines to read.
  {
    const int chunks = half / E, n = 2 * c.kv_heads * chunks * 16;
#pragma unroll 2
    for (int i = work; i < n; i += stride) {
      const int y = i >> 4, d = y % chunks * E, x = y / chunks, h = x % c.kv_heads;
      const int t = base + (x / c.kv_heads) * 16 + (i & 15) - low;
      if (t < 0 || t >= count) continue;
      alignas(16) float lo[E], hi[E];
      load(k + (size_t(row0 + t) * c.kv_heads + h) * dim, t, d, lo, hi);
      alignas(16) T out[2][E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        out[0][e] = T(lo[e]);
        out[1][e] = T(hi[e]);
      }
      T *dst = pages + h * head;
      *reinterpret_cast<uint4 *>(dst + dev::key_place<E>(t_low + t, d, dim)) = *reinterpret_cast<const uint4 *>(out[0]);
      *reinterpret_cast<uint4 *>(dst + dev::key_place<E>(t_low + t, d + half, dim)) =
          *reinterpret_cast<const uint4 *>(out[1]);
    }
  }
  // v: a channel of a piece of E tokens per thread (16 a + 4 piece + b of the
  // group, or 4 piece + b).
  constexpr int pieces = kAppendGroup / E;
  const int n = c.kv_heads * pieces * dim;
#pragma unroll 2
  for (int i = work; i < n; i += stride) {
    const int d = i % dim, y = i / dim, piece = y % pieces, h = y / pieces;
    auto token = [&](int e) { return E == 8 ? (e >> 2) * 16 + 4 * piece + (e & 3) : 4 * piece + e; };
    alignas(16) T out[E];
    int have = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int t = base + token(e) - low;
      const bool in = t >= 0 && t < count;
      have += in;
      out[e] = T(in ? v[(size_t(row0 + t) * c.kv_heads + h) * dim + d] : 0.0f);
    }
    T *dst = pages + (c.kv_heads + h) * head + dev::value_place<E>((base & (c.page_size - 1)) + token(0), d, dim);
    if (have == E) {
      *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(out);
    } else if (have) {  // the piece's other tokens stay
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int t = base + token(e) - low;
        if (t >= 0 && t < count) dst[e] = out[e];
      }
    }
  }
}

__global__ void k_paged_advance(int *lengths, const PagedBatch b) {
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s >= b.sequences) return;
  int first, end;
  dev::row_range(b, s, first, end);
  const int limit = b.table_pages << b.page_shift, length = min(max(lengths[s], 0), limit), grown = length + end - first;
  if (grown > limit || length != lengths[s]) atomicOr(b.err, kPagedErr);
  lengths[s] = min(grown, limit);
}

// ---------------------------------------------------------------------------
// Reorder: every sequence takes the keys of its parent in the same group.  All
// of a group have one length.  Full pages are only read from now on, so
// children share them: their table columns are copied.  The partial page is
// written to next, so each child needs its own: a parent's first child (in
// slot order) takes the parent's page over, further children get the pages of
// parents without children, in ascending order, and a copy of what is in them.
// No page that is copied from is copied to, and the old tables are only read:
// one launch does both, and doing it again gives the same.  Later columns stay.
constexpr int kReorderThreads = 256;
constexpr int kReorderMaxShare = 64;

__global__ __launch_bounds__(kReorderThreads) void k_paged_reorder(int *new_tables, const PagedBatch b,
                                                                   const int *parents, const PagedLayers layers,
                                                                   const PagedCache c, int pairs, int write_tables) {
  __shared__ int parent[kReorderMaxShare], target[kReorderMaxShare], page_of[kReorderMaxShare], again_of[kReorderMaxShare];
  __shared__ int partial_page[kReorderMaxShare];
  __shared__ int ok, extra;
  const int group = blockIdx.x / pairs, pair = blockIdx.x % pairs, tid = threadIdx.x;
  const int s0 = group * b.share, runs = 2 * c.kv_heads;
  // Parents and lengths are on their way together, the page ids of the partly
  // filled pages as soon as the length is there.
  const bool in = tid < b.share;
  const int wanted = in ? parents[s0 + tid] : 0, own = in ? b.lengths[s0 + tid] : 0;
  const int length = dev::own_length(b, s0), full = length >> b.page_shift, rest = length & (c.page_size - 1);
  const bool tables = int(blockIdx.z) == runs;
  if (tables ? !write_tables || pair != 0 || blockIdx.y != 0 : rest == 0) return;
  if (tid < 64) {  // one wave plans the group
    const int id = in && rest ? b.tables[size_t(s0 + tid) * b.table_pages + full] : 0;
    const int p = in ? wanted - s0 : -1;
    const bool bad = in && (unsigned(p) >= unsigned(b.share) || own != length);
    if (in) parent[tid] = bad ? tid : p;
    const bool all = __ballot(bad) == 0;
    if (bad) atomicOr(b.err, kPagedErr);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    bool again = false, has_child = false;
    for (int j = 0; j < b.share; ++j) {
      again |= j < tid && parent[j] == p;
      has_child |= parent[j] == tid;
    }
    again &= in && all;
    const bool free = in && all && !has_child;
    const uint64_t before = (uint64_t(1) << tid) - 1;
    const uint64_t again_mask = __ballot(again), free_mask = __ballot(free);
    if (free) target[__popcll(free_mask & before)] = tid;
    if (again) again_of[__popcll(again_mask & before)] = tid;
    if (in) page_of[tid] = again ? -1 - __popcll(again_mask & before) : p;  // whose page a slot takes
    if (in) partial_page[tid] = id;
    if (tid == 0) {
      ok = all;
      extra = __popcll(again_mask);
    }
  }
  __syncthreads();
  if (tables) {
    for (int i = tid; i < b.share * b.table_pages; i += kReorderThreads) {
      const int slot = i / b.table_pages, col = i % b.table_pages;
      int from = slot;
      if (ok && col < full) from = parent[slot];
      if (ok && col == full && rest) from = page_of[slot] < 0 ? target[-1 - page_of[slot]] : page_of[slot];
      new_tables[size_t(s0) * b.table_pages + i] = b.tables[size_t(s0 + from) * b.table_pages + col];
    }
    return;
  }
  if (!ok || pair >= extra) return;
  const int from = dev::checked_page(partial_page[parent[again_of[pair]]], b);
  const int to = dev::checked_page(partial_page[target[pair]], b);
  if (from < 0 || to < 0) return;
  const size_t run = size_t(c.page_size) * c.dim * (c.bf16 ? 2 : 4), page = run * runs;
  const int pieces = (rest + 31) / 32 * 32 * c.dim * (c.bf16 ? 2 : 4) / 16;
  uint8_t *base = static_cast<uint8_t *>(layers.pages[blockIdx.y]) + blockIdx.z * run;
  const uint4 *src = reinterpret_cast<const uint4 *>(base + from * page);
  uint4 *dst = reinterpret_cast<uint4 *>(base + to * page);
  for (int i = tid; i < pieces; i += kReorderThreads) dst[i] = src[i];
}

// Rows of 32-bit words by index; an index outside gives zeros and the error word.
__global__ __launch_bounds__(256) void k_gather_rows(uint32_t *dst, const uint32_t *src, const int *indices, int rows,
                                                     int cols, int src_rows, int *err) {
  for (unsigned r = blockIdx.x; r < unsigned(rows); r += gridDim.x) {
    const int from = indices[r];
    const bool ok = unsigned(from) < unsigned(src_rows);
    if (!ok && threadIdx.x == 0) atomicOr(err, kPagedErr);
    // (unsigned: a row may end less than a step below 2^31)
    for (unsigned i = blockIdx.y * 256 + threadIdx.x; i < unsigned(cols); i += gridDim.y * 256)
      dst[size_t(r) * cols + i] = ok ? src[size_t(from) * cols + i] : 0u;
  }
}

}  // namespace

void paged_append_launch(const PagedCache &c, const PagedBatch &b, const float *k, const float *v, const float *q,
                         float *q_out, int heads, float theta, hipStream_t s) {
  // Groups from two rows per sequence on.  9 ragged prompts, 1501 rows of 32
  // and 8 heads, 128 channels: 53 us with workgroups per row, 41 in groups.
  if (b.starts && b.rows >= 2 * b.sequences) {
    const int groups = b.rows / kAppendGroup + 2 * b.sequences;
    const dim3 grid(groups + report_groups(b), std::max(1, std::min(16, 4096 / groups)));
    const size_t lds = size_t(kAppendGroup) * c.dim / 2 * sizeof(double2);
    if (c.bf16)
      k_paged_append_groups<8, __bf16><<<grid, kAppendThreads, lds, s>>>(c, b, k, v, q, q_out, heads, theta);
    else
      k_paged_append_groups<4, float><<<grid, kAppendThreads, lds, s>>>(c, b, k, v, q, q_out, heads, theta);
    hip_check(hipGetLastError(), "paged append launch");
    return;
  }
  const int items = ((q ? heads : 0) + 3 * c.kv_heads) * c.dim / 2;
  const dim3 grid(b.rows + report_groups(b), std::min((items + kAppendThreads - 1) / kAppendThreads, b.rows < 64 ? 16 : 2));
  if (c.bf16)
    k_paged_append<8, __bf16><<<grid, kAppendThreads, 0, s>>>(c, b, k, v, q, q_out, heads, theta);
  else
    k_paged_append<4, float><<<grid, kAppendThreads, 0, s>>>(c, b, k, v, q, q_out, heads, theta);
  hip_check(hipGetLastError(), "paged append launch");
}

void paged_advance_launch(int *lengths, const PagedBatch &b, hipStream_t s) {
  k_paged_advance<<<(b.sequences + 255) / 256, 256, 0, s>>>(lengths, b);
  hip_check(hipGetLastError(), "paged advance launch");
}

void paged_reorder_launch(int *new_tables, const PagedBatch &b, const int *parents, const PagedLayers &layers, int count,
                          const PagedCache &shape, bool write_tables, hipStream_t s) {
  const int pairs = std::max(1, b.share - 1);
  const dim3 grid(b.sequences / b.share * pairs, count, 2 * shape.kv_heads + 1);
  k_paged_reorder<<<grid, kReorderThreads, 0, s>>>(new_tables, b, parents, layers, shape, pairs, write_tables);
  hip_check(hipGetLastError(), "paged reorder launch");
}

void gather_rows_launch(float *dst, const float *src, const int *indices, int rows, int cols, int src_rows, int *err,
                        hipStream_t s) {
  // (A launch counts its threads along x in 32 bits.)
  const dim3 grid(std::min(rows, 1 << 22), std::min((cols - 1) / 1024 + 1, 64));
  k_gather_rows<<<grid, 256, 0, s>>>(reinterpret_cast<uint32_t *>(dst), reinterpret_cast<const uint32_t *>(src), indices,
                                     rows, cols, src_rows, err);
  hip_check(hipGetLastError(), "gather rows launch");
}

}  // namespace qnn
