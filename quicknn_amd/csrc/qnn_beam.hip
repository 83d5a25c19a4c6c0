// qnn_beam.hip -- the best continuations of beams: per group, the `select`
// largest of score[b] + log_softmax(logits[b])[v] over beams and vocabulary.
//
// One pass over the logits leaves every tile's maximum and sum of exponentials
// (a wave per tile of 64 to 1024 tokens).  The second launch, a workgroup per
// group, joins the sums and takes T, the select-th largest of the tiles' best
// candidates: `select` candidates reach T, so nothing below T is among the
// result, and only tiles whose best reaches T (`select` of them, but for ties)
// are read again.  What reaches T there, a few times `select` candidates, is
// ranked by counting.  The tile is chosen small enough that a group has several
// times `select` of them, down to a wave's width.  Where more than 512 reach T
// (ties: flat logits, or logits masked with a large finite value, all of which
// round to one fp32 candidate; or `select` near 64, where the bound behind T is
// the least of a wave's maxima), every wave keeps its best in order in one more
// pass, and their lists are ranked: 8 groups of 8 beams over 151936 masked
// tokens, 16 selected, 490 us; 4 groups of 32 beams over 32000, 64 selected, 600
// us (11.4 and 25 ms with a pass over all of them per rank).
//
// Candidates are compared in 64 bits.  Logits of one beam are exact there; two
// beams' normalisers carry the roundings of fp32 sums, so the order across
// beams is that of the exact values but for gaps of about 1e-7.  Equal logits
// give equal sums, whatever their rows' alignment.  The scores are rounded to
// fp32 once.
//
// What bounds it: the first launch memory (38.9 MB of logits in 8 us), the
// second one chain of latencies in one workgroup per group (12 us for 8 groups
// of 8 beams over 151936 tokens, select 16; 8 us for 4 beams over 32000).  A
// ranked list per 4096-token tile in the first launch and a merge of the lists
// by rounds took 20 and 38 us.
#include <cmath>

#include "qnn_internal.h"
#include "qnn_lanes.h"
#include "qnn_topk_dev.h"

namespace qnn {
namespace {

constexpr int kScanThreads = 256, kMergeThreads = 1024;
constexpr int kPerLaneMax = 16;
constexpr int kList = 4096;  // tiles read again and candidates in LDS, at most; with more (ties) all tiles are looked at
constexpr float kLog2e = 1.4426950408889634f;

struct TileStat {
  float top, sum;  // the largest logit; the sum of exp(logit - top), NaN with a NaN or plus infinity in the tile
};

template <int E>  // tokens per lane
__global__ __launch_bounds__(kScanThreads) void k_beam_scan(const BeamArgs a, int tiles, TileStat *stats) {
  const int beam = blockIdx.y, lane = threadIdx.x & 63, tile = blockIdx.x * (kScanThreads / 64) + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const float *row = a.logits + size_t(beam) * a.vocab;
  const unsigned item = unsigned(tile) * (64 * E) + lane, end = unsigned(a.vocab) - 1u;
  float x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = __builtin_nontemporal_load(row + min(item + unsigned(i) * 64, end));
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (item + unsigned(i) * 64 > end) x[i] = -INFINITY;
    top = fmaxf(top, x[i]);
  }
  top = dev::wave_max_xor(top);
  const float zero = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) sum += __builtin_amdgcn_exp2f((x[i] - zero) * kLog2e);
  sum = dev::wave_sum_xor(sum);
  if (lane == 0) stats[size_t(beam) * tiles + tile] = {top, sum};
}

// What a beam's tokens are.
enum Kind { kLive, kDone, kNone };

struct Merge {
  double lse[kBeamMax], score[kBeamMax];
  int kind[kBeamMax];
  unsigned bound[kMergeThreads / 64], limit;
  int tiles, found;       // counts of the lists
  int kept;
  int list[kList];
  unsigned key[kList];
  double value[kList];
  unsigned flat[kList];
};

template <int OFF>
__device__ __forceinline__ double xor_lanes(double x) {
  return __hiloint2double(dev::xor_lanes_i<OFF>(__double2hiint(x)), dev::xor_lanes_i<OFF>(__double2loint(x)));
}
__device__ __forceinline__ double wave_sum(double x) {
  x += xor_lanes<32>(x);
  x += xor_lanes<16>(x);
  x += xor_lanes<8>(x);
  x += xor_lanes<4>(x);
  x += xor_lanes<2>(x);
  return x + xor_lanes<1>(x);
}

__device__ __forceinline__ bool before(double v, unsigned f, double w, unsigned g) { return v > w || (v == w && f < g); }

__global__ __launch_bounds__(kMergeThreads) void k_beam_merge(const BeamArgs a, int tiles, int per_lane,
                                                              const TileStat *stats) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  Merge &sh = *reinterpret_cast<Merge *>(lds);
  const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = group * a.beams;
  const TileStat *mine = stats + size_t(first) * tiles;
  // ---- each beam's normaliser, a wave per beam
  for (int b = wave; b < a.beams; b += kMergeThreads / 64) {
    const TileStat *st = mine + size_t(b) * tiles;
    const float score = a.scores[first + b];
    const bool done = a.done && a.done[first + b];
    float own = -INFINITY;  // a lane's tiles, four on their way at once
    double sum = 0.0;
    for (int t0 = lane; t0 < tiles; t0 += 256) {
      TileStat x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = st[min(t0 + j * 64, tiles - 1)];
      const float old = own;
#pragma unroll
      for (int j = 0; j < 4; ++j) own = fmaxf(own, x[j].top);
      const float zero = own == -INFINITY ? 0.0f : own;
      sum *= double(__builtin_amdgcn_exp2f((old - zero) * kLog2e));
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (t0 + j * 64 < tiles) sum += double(x[j].sum) * double(__builtin_amdgcn_exp2f((x[j].top - zero) * kLog2e));
    }
    const float top = dev::wave_max_xor(own);
    sum *= double(__builtin_amdgcn_exp2f((own - (top == -INFINITY ? 0.0f : top)) * kLog2e));
    sum = wave_sum(sum);
    if (lane == 0) {
      sh.lse[b] = double(top) + log(sum);
      sh.score[b] = score;
      sh.kind[b] = !isfinite(score) ? kNone : done ? kDone : sum != sum || !isfinite(top) ? kNone : kLive;
    }
  }
  if (tid == 0) sh.tiles = sh.found = sh.kept = 0;
  __syncthreads();
  auto candidate = [&](int b, float logit) { return sh.score[b] + (double(logit) - sh.lse[b]); };
  // The order bits of tile i's best candidate rounded to fp32 (rounding keeps
  // the order); 0 where it has none above minus infinity.  A beam that is done
  // has one, in its first tile.
  auto best_of = [&](int i) -> unsigned {
    const int b = i / tiles, t = i - b * tiles;
    double c = -INFINITY;
    if (sh.kind[b] == kLive) c = candidate(b, mine[i].top);
    else if (sh.kind[b] == kDone && t == 0) c = sh.score[b];
    return c == -INFINITY ? 0u : dev::order_bits(float(c));
  };
  // ---- T.  First a bound: of a wave's 64 thread maxima, the largest value that
  // `select` reach (found bit by bit, by ballots, no barrier); the largest of
  // the waves'.  The tiles that reach it are listed; if they are few, T is the
  // select-th largest of theirs, by counting.  (Four byte-wise radix passes
  // with their 13 barriers took 2 us longer.)
  const int n = a.beams * tiles;
  constexpr int kKept = 2;  // of a thread's tiles; further ones are computed twice
  unsigned kept[kKept], most = 0;
#pragma unroll
  for (int r = 0; r < kKept; ++r) {
    const int i = tid + r * kMergeThreads;
    kept[r] = i < n ? best_of(i) : 0u;
    most = max(most, kept[r]);
  }
  for (int i = tid + kKept * kMergeThreads; i < n; i += kMergeThreads) most = max(most, best_of(i));
  unsigned bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned c = bound | 1u << bit;
    if (__popcll(__ballot(most >= c)) >= a.select) bound = c;
  }
  if (lane == 0) sh.bound[wave] = bound;
  __syncthreads();
  bound = 1;  // (below that: no candidate)
  for (int w = 0; w < kMergeThreads / 64; ++w) bound = max(bound, sh.bound[w]);
  auto list = [&](int i, unsigned k) {
    if (k >= bound) {
      const int at = atomicAdd(&sh.tiles, 1);
      if (at < kList) sh.list[at] = i, sh.key[at] = k;
    }
  };
#pragma unroll
  for (int r = 0; r < kKept; ++r) list(tid + r * kMergeThreads, kept[r]);
  for (int i = tid + kKept * kMergeThreads; i < n; i += kMergeThreads) list(i, best_of(i));
  __syncthreads();
  int count = sh.tiles;
  if (count > a.select && count <= 512) {
    unsigned k = 0;
    int i = 0;
    if (tid < count) {
      k = sh.key[tid];
      i = sh.list[tid];
      int above = 0, same = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j) {
        above += sh.key[j] > k;
        same += sh.key[j] == k;
      }
      if (above < a.select && above + same >= a.select) sh.limit = k;  // from all that are equal, the same
    }
    __syncthreads();
    bound = sh.limit;
    if (k >= bound) sh.list[atomicAdd(&sh.kept, 1)] = i;  // (every thread has read its own)
    __syncthreads();
    count = sh.kept;
  }
  const unsigned limit = bound;
  // (Unsigned from here: the last tile may end behind 2^31.)
  const unsigned span = 64 * per_lane, vocab = a.vocab;
  // The candidate of token v of beam b.
  auto value_of = [&](int b, int v) -> double {
    if (sh.kind[b] == kLive) return candidate(b, a.logits[size_t(first + b) * a.vocab + v]);
    return sh.kind[b] == kDone && v == a.end ? sh.score[b] : -INFINITY;
  };
  auto reaches = [&](double c) { return c > -INFINITY && dev::order_bits(float(c)) >= limit; };
  if (count <= kList)
    for (int x = wave; x < count; x += kMergeThreads / 64) {
      // (The list has run over: the tiles are read again below.)
      if (__hip_atomic_load(&sh.found, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP) > kList) break;
      const int i = sh.list[x], b = i / tiles, t = i - b * tiles;
      if (sh.kind[b] == kDone) {
        if (lane == 0) {
          const int at = atomicAdd(&sh.found, 1);
          if (at < kList) sh.value[at] = sh.score[b], sh.flat[at] = b * vocab + a.end;
        }
        continue;
      }
      // All of the tile is requested at once (one by one, a chain of loads: 5 us more).
      const float *row = a.logits + size_t(first + b) * a.vocab;
      float y[kPerLaneMax];
#pragma unroll
      for (int j = 0; j < kPerLaneMax; ++j) y[j] = row[min(t * span + min(j, per_lane - 1) * 64 + lane, vocab - 1)];
#pragma unroll
      for (int j = 0; j < kPerLaneMax; ++j) {
        const unsigned v = t * span + j * 64 + lane;
        const double c = j < per_lane && v < vocab ? candidate(b, y[j]) : -INFINITY;
        if (reaches(c)) {
          const int at = atomicAdd(&sh.found, 1);
          if (at < kList) sh.value[at] = c, sh.flat[at] = b * vocab + v;
        }
      }
    }
  __syncthreads();
  const int found = count <= kList ? sh.found : kList + 1;
  auto put = [&](int rank, double c, unsigned flat) {
    const size_t at = size_t(group) * a.select + rank;
    a.parents[at] = first + int(flat / vocab);
    a.tokens[at] = int(flat % vocab);
    a.best[at] = float(c);
  };
  int ranked = min(found, a.select), entries = found;
  if (found > 512) {
    // Many (ties, flat or masked logits, few tiles): one more pass, from the
    // list or, if that ran over, over all that reach T.  Every wave keeps the
    // best 64 of its share, one per lane in order; their lists are ranked below.
    ranked = a.select;
    entries = a.select * (kMergeThreads / 64);
    double c = -INFINITY;
    unsigned f = ~0u;
    auto offer = [&](double c1, unsigned f1) {  // a candidate per lane, minus infinity for none
      const double cw = __shfl(c, a.select - 1);
      const unsigned fw = __shfl(f, a.select - 1);
      uint64_t in = __ballot(c1 > -INFINITY && before(c1, f1, cw, fw));
      for (; in; in &= in - 1) {
        const int from = __ffsll(static_cast<unsigned long long>(in)) - 1;
        const double c2 = __shfl(c1, from), above_c = __shfl_up(c, 1);
        const unsigned f2 = __shfl(f1, from), above_f = __shfl_up(f, 1);
        const int at = __popcll(__ballot(before(c, f, c2, f2)));
        if (lane > at) c = above_c, f = above_f;
        else if (lane == at) c = c2, f = f2;
      }
    };
    auto offer_tile = [&](int i) {
      const int b = i / tiles, t = i - b * tiles;
      if (sh.kind[b] == kDone) {
        offer(lane == 0 ? sh.score[b] : -INFINITY, b * vocab + a.end);
        return;
      }
      const float *row = a.logits + size_t(first + b) * a.vocab;
      for (int j0 = 0; j0 < per_lane; j0 += 8) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = row[min(t * span + min(j0 + j, per_lane - 1) * 64 + lane, vocab - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned v = t * span + (j0 + j) * 64 + lane;
          const double c1 = j0 + j < per_lane && v < vocab ? candidate(b, y[j]) : -INFINITY;
          offer(reaches(c1) ? c1 : -INFINITY, b * vocab + v);
        }
      }
    };
    if (found <= kList) {
      for (int j0 = wave * 64; j0 < found; j0 += kMergeThreads) {
        const int j = min(j0 + lane, found - 1);
        offer(j0 + lane < found ? sh.value[j] : -INFINITY, sh.flat[j]);
      }
    } else if (count <= kList) {
      for (int x = wave; x < count; x += kMergeThreads / 64) offer_tile(sh.list[x]);
    } else {
      for (int i = wave; i < n; i += kMergeThreads / 64)
        if (best_of(i) >= limit) offer_tile(i);
    }
    __syncthreads();  // the lists have been read
    if (lane < a.select) {
      sh.value[wave * a.select + lane] = c;
      sh.flat[wave * a.select + lane] = f;
    }
    __syncthreads();
  }
  if (tid < entries) {
    const double c = sh.value[tid];
    const unsigned f = sh.flat[tid];
    int rank = 0;
    for (int j = 0; j < entries; ++j) rank += before(sh.value[j], sh.flat[j], c, f);
    if (c > -INFINITY && rank < a.select) put(rank, c, f);
  }
  // ---- fewer candidates than ranks: minus infinities in order.  (All finite
  // ones are taken then, less than `select`, so nearly every token is one.)
  if (ranked < a.select && wave == 0) {
    const unsigned all = a.beams * vocab;
    for (unsigned f0 = 0; ranked < a.select && f0 < all; f0 += 64) {
      const unsigned f = f0 + lane;
      const bool in = f < all && value_of(int(f / vocab), int(f % vocab)) == -INFINITY;
      const uint64_t mask = __ballot(in);
      const int rank = ranked + __popcll(mask & ((uint64_t(1) << lane) - 1));
      if (in && rank < a.select) put(rank, -INFINITY, f);
      ranked += __popcll(mask);
    }
  }
}

// Tokens per lane: the most that leaves a group 8 tiles per selected candidate.
int per_lane_of(const BeamArgs &a) {
  int e = kPerLaneMax;
  while (e > 1 && int64_t(a.beams) * a.vocab / (64 * e) < 8 * a.select) e /= 2;
  return e;
}
int tiles_of(const BeamArgs &a) { return (a.vocab - 1) / (64 * per_lane_of(a)) + 1; }

}  // namespace

size_t beam_select_bytes(const BeamArgs &a) { return size_t(a.groups) * a.beams * tiles_of(a) * sizeof(TileStat); }

void beam_select_launch(const BeamArgs &a, void *ws, hipStream_t s) {
  const int e = per_lane_of(a), tiles = tiles_of(a);
  TileStat *stats = static_cast<TileStat *>(ws);
  const dim3 grid((tiles + kScanThreads / 64 - 1) / (kScanThreads / 64), a.groups * a.beams);
  switch (e) {
    case 1: k_beam_scan<1><<<grid, kScanThreads, 0, s>>>(a, tiles, stats); break;
    case 2: k_beam_scan<2><<<grid, kScanThreads, 0, s>>>(a, tiles, stats); break;
    case 4: k_beam_scan<4><<<grid, kScanThreads, 0, s>>>(a, tiles, stats); break;
    case 8: k_beam_scan<8><<<grid, kScanThreads, 0, s>>>(a, tiles, stats); break;
    default: k_beam_scan<kPerLaneMax><<<grid, kScanThreads, 0, s>>>(a, tiles, stats); break;
  }
  hip_check(hipGetLastError(), "beam scan launch");
  hip_check(hipFuncSetAttribute(reinterpret_cast<const void *>(k_beam_merge), hipFuncAttributeMaxDynamicSharedMemorySize,
                                int(sizeof(Merge))),
            "beam merge LDS size");
  k_beam_merge<<<a.groups, kMergeThreads, sizeof(Merge), s>>>(a, tiles, e, stats);
  hip_check(hipGetLastError(), "beam merge launch");
}

}  // namespace qnn
