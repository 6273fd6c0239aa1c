// The paged cache's row and slot operators on gfx950: norm, rotation and
// store of new rows (lfm3_paged_heads) and the eviction by accumulated weight
// (lfm3_paged_evict).
#include <algorithm>

#include "paged.hpp"

namespace lfm3amd {
namespace {

// ------------------------------------------------------------------- heads

struct HeadsArgs {
  const float *q, *k, *v;
  std::size_t ld;
  const float *q_norm, *k_norm, *frequencies, *factors;
  void* q_out;
  std::size_t ldq;
  Half *k_pages, *v_pages;
  float* weight;
  PageTable table;
  const std::uint32_t *starts, *lengths, *positions;
  int seqs, heads, kv_heads;
  float eps;
  std::uint32_t first_row;  // of the launch
};

// The sequence of a row: the number of starts[1 ..] at or before it. Lanes
// read 64 starts at a time, so a batch's search is one memory round trip.
__device__ __forceinline__ int SequenceOf(const std::uint32_t* starts, int seqs, std::uint32_t row,
                                          int lane) {
  int seq = 0;
  for (int base = 0; base < seqs; base += 64)
    seq += __popcll(__ballot(base + lane < seqs && starts[base + lane + 1] <= row));
  return __builtin_amdgcn_readfirstlane(seq);
}

// x normed over its D values and rotated: a thread holds the pair (i, i + D /
// 2) of a head, D / 2 threads a head. RMSNorm scale = 1 / sqrt(mean(x^2) +
// eps); the pair (a, b) turns to (a cos - b sin, b cos + a sin).
template<int D>
__device__ __forceinline__ float HeadSum(float v) {
  v = SumXor16(GroupSum16(v));
  return D == 128 ? SumXor32(v) : v;
}

// A thread's pair of one unit (query heads, then keys, then values), D / 2
// threads a unit; each forms its own angle and takes it into [-pi, pi] in FP64: in
// FP32 position * frequency alone is off by up to 4e-3 radians at position 131072.
// Bound by the launch and two dependent reads before the first store: 8 rows of 24
// heads of 128 3.0 to 3.3 us; 519 rows of 48 heads of 64 (9.5 MB) 6.0 to 6.4 us,
// 1.5 TB/s, where a launch (3) and the bytes (2) are 5.
template<int D, class T, bool kRows32>
__launch_bounds__(256) __global__ void PagedHeadsKernel(HeadsArgs a) {
  constexpr int P = D / 2, kParts = 256 / P;
  const int tid = threadIdx.x, pair = tid % P, part = tid / P;
  const std::uint32_t row = a.first_row + blockIdx.x;
  const int seq = SequenceOf(a.starts, a.seqs, row, tid & 63);
  if (seq >= a.seqs || row < a.starts[seq])
    return;
  const std::uint32_t first = a.starts[seq], n = a.starts[seq + 1] - first, ahead = row - first;
  const std::uint32_t length = a.lengths[seq];
  const bool held = length >= n;
  const std::uint32_t slot = length - n + ahead;
  const std::uint32_t page = held ? a.table.Page(seq, slot) : ~0u;
  const bool stored = page < a.table.pages;
  const int page_slots = 1 << a.table.shift;
  const double position = double(a.positions[seq]) + double(ahead);
  double angle = position * double(a.frequencies[pair]);
  if (a.factors)
    angle /= double(a.factors[pair]);
  constexpr double kTurn = 6.283185307179586476925;
  float sn, cs;
  sincosf(float(angle - kTurn * rint(angle * (1.0 / kTurn))), &sn, &cs);
  const int u = blockIdx.y * kParts + part;
  if (u >= a.heads + 2 * a.kv_heads)
    return;
  const bool is_q = u < a.heads, is_k = !is_q && u < a.heads + a.kv_heads;
  const int g = is_q ? u : is_k ? u - a.heads : u - a.heads - a.kv_heads;
  const float* x = (is_q ? a.q : is_k ? a.k : a.v) + row * a.ld + std::size_t(g) * D;
  const float x0 = x[pair], x1 = x[pair + P];
  float r0 = x0, r1 = x1;
  if (is_q || is_k) {
    const float* w = is_q ? a.q_norm : a.k_norm;
    const float inv = 1.0f / sqrtf(HeadSum<D>(x0 * x0 + x1 * x1) / float(D) + a.eps);
    const float y0 = (x0 * inv) * w[pair], y1 = (x1 * inv) * w[pair + P];
    r0 = y0 * cs - y1 * sn;
    r1 = y1 * cs + y0 * sn;
  }
  if (is_q) {
    const std::size_t at = row * a.ldq + std::size_t(g) * D + pair;
    StoreRow<T, kRows32>(a.q_out, at, r0);
    StoreRow<T, kRows32>(a.q_out, at + P, r1);
  } else if (stored) {
    const std::size_t cell =
        (std::size_t(page) * a.kv_heads + g) * page_slots + (slot & (page_slots - 1));
    Half* pool = is_k ? a.k_pages : a.v_pages;
    pool[cell * D + pair] = T::Round(r0);
    pool[cell * D + pair + P] = T::Round(r1);
    if (is_k && a.weight && pair == 0)
      a.weight[cell] = 0.0f;
  }
}

// Blocks of a launch in x: a grid has less than 2^32 threads there.
constexpr std::uint32_t kMaxBlocks = 1u << 23;

template<int D, class T>
void LaunchHeads(HeadsArgs a, std::uint32_t rows, std::uint32_t units, bool rows32,
                 hipStream_t s) {
  constexpr std::uint32_t kParts = 512 / D;
  for (; a.first_row < rows; a.first_row += kMaxBlocks) {
    const dim3 grid(std::min(rows - a.first_row, kMaxBlocks), (units + kParts - 1) / kParts);
    if (rows32)
      PagedHeadsKernel<D, T, true><<<grid, 256, 0, s>>>(a);
    else
      PagedHeadsKernel<D, T, false><<<grid, 256, 0, s>>>(a);
  }
}

// ------------------------------------------------------------------- evict

// A weight's rank: its bits made monotone as unsigned, NaN above all, -0 as 0.
// 0 is left for slots on no page.
__device__ __forceinline__ unsigned RankOf(float w) {
  if (w != w)
    return 0xffffffffu;
  const unsigned bits = __float_as_uint(w + 0.0f);
  return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}

struct EvictArgs {
  Half *k_pages, *v_pages;
  float* weight;
  PageTable table, new_table;
  const std::uint32_t* lengths;
  std::uint32_t max_length, budget, sinks, recent;
  std::uint32_t* kept;
  unsigned* counts;  // of each list's kept slots; NULL: the move finds them again
  int kv_heads;
};

// What a sequence keeps: its first `lo` slots, those from `hi` on, and of those
// between that lie on a page up to `need`.
struct EvictRange {
  std::uint32_t length, lo, hi, need;
  __device__ __forceinline__ EvictRange(const EvictArgs& a, int seq) {
    length = min(a.lengths[seq], a.max_length);
    lo = min(a.sinks, length);
    hi = max(lo, length - min(a.recent, length));
    need = a.budget - a.sinks - a.recent;
  }
  // Slots kept in all, `ranked` of them between lo and hi.
  __device__ __forceinline__ std::uint32_t Count(std::uint32_t ranked) const {
    return lo + ranked + (length - hi);
  }
};

// A thread's share of the number of a sequence's slots [from, to) that lie on a
// page.
__device__ __forceinline__ unsigned PresentShare(const PageTable& table, int seq,
                                                 std::uint32_t from, std::uint32_t to,
                                                 int threads) {
  unsigned n = 0;
  if (from < to)
    for (std::uint32_t e = (from >> table.shift) + threadIdx.x; e <= (to - 1) >> table.shift;
         e += threads)
      if (table.Page(seq, e << table.shift) < table.pages)
        n += min(to, (e + 1) << table.shift) - max(from, e << table.shift);
  return n;
}
// The sum of every thread's v in all threads; s_wave: a word a wave.
template<int kWaves>
__device__ __forceinline__ unsigned BlockTotal(unsigned v, unsigned* s_wave) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0)
    s_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  unsigned total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    total += s_wave[w];
  __syncthreads();
  return total;
}

// Workspace of an eviction in slices (LaunchSlices).
struct EvictSlices {
  unsigned* ranks;   // [seq][head][slices * slice]
  unsigned* bins;    // [digit][seq][head][slices][kBins]
  uint2* state;      // [digit][seq][head]: the prefix so far, and what is needed of it
  unsigned* above;   // [seq][head][slices]: slots of earlier slices that rank above it
  std::uint32_t slice, slices;
};

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kDigitBits = 11, kBins = 1 << kDigitBits;
// Up to so many slots one block finds a list, their ranks in its LDS; beyond,
// slices of at least kSlice slots, at most kMaxSlices of them, and of twice as
// many where those are more than the CUs (128 lists of 32,760 slots 79 us, 105 in
// slices of 4096; 8 of 65,536 36 us, 38 in slices of 8192). With the move, one
// block and slices: 32 lists of 8190 slots 32 and 39 us, of 16,000 44 and 40, 160
// lists of 16,000 47 and 73; 32 of 24,000 53 and 42, 8 of 32,760 57 and 32.
constexpr std::uint32_t kOneBlock = 16384, kSlice = 4096, kMaxSlices = 32,
                        kCus = 256;

// Rank of a slot's weight.
__device__ __forceinline__ unsigned ReadRank(const EvictArgs& a, int seq, int g,
                                             std::uint32_t slot) {
  const int page_slots = 1 << a.table.shift;
  const std::uint32_t page = a.table.Page(seq, slot);
  const float w =
      a.weight[(std::size_t(page < a.table.pages ? page : 0u) * a.kv_heads + g) * page_slots +
               (slot & (page_slots - 1))];
  return page < a.table.pages ? RankOf(w) : 0u;
}

// A digit of the threshold. Digit 0: bits 21..31, 1: 10..20, 2: 0..9.
struct Digit {
  int low, bits;
  __device__ __forceinline__ explicit Digit(int d)
      : low(d == 0 ? 21 : d == 1 ? 10 : 0), bits(d == 2 ? 10 : kDigitBits) {}
  // The bits of the digits before this one.
  __device__ __forceinline__ unsigned Before() const {
    return low + bits == 32 ? 0u : ~0u << (low + bits);
  }
  __device__ __forceinline__ unsigned Bin(unsigned rank) const {
    return (rank >> low) & ((1u << bits) - 1);
  }
};

// The bin that holds the need-th slot from the top of a histogram of which
// thread i holds bins 2047 - 2 i (x0) and the one below (x1); bins that a digit
// does not have are empty. s_total: a word a wave, s_pick: two. Every thread
// gets the bin and what is needed of it; ends with a barrier passed.
__device__ __forceinline__ uint2 FindBin(unsigned x0, unsigned x1, unsigned need, unsigned* s_total,
                                         unsigned* s_pick) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  unsigned run = x0 + x1;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned up = __shfl_up(run, d);
    run += lane >= d ? up : 0u;
  }
  if (lane == 63)
    s_total[wave] = run;
  __syncthreads();
  unsigned above = run - x0 - x1;
  for (int w = 0; w < wave; ++w)
    above += s_total[w];
  if (above < need && need <= above + x0 + x1) {
    const bool lower = need > above + x0;
    s_pick[0] = unsigned(kBins - 1 - 2 * tid - (lower ? 1 : 0));
    s_pick[1] = need - above - (lower ? x0 : 0u);
  }
  __syncthreads();
  return make_uint2(s_pick[0], s_pick[1]);
}

// Where the ranked slots are cut: those of a rank above `prefix` are kept and the
// first `need` of rank `prefix`, `ranked` in all.
struct Cut {
  unsigned prefix, need, ranked;
  // wanted: slots asked for; prefix, need: the last one's rank, and what is
  // needed of it (nothing of rank 0, which is on no page).
  static __device__ __forceinline__ Cut At(unsigned wanted, unsigned prefix, unsigned need) {
    if (!wanted)
      return Cut{0xffffffffu, 0, 0};
    return prefix ? Cut{prefix, need, wanted} : Cut{0, 0, wanted - need};
  }
  // All that lie on a page, of which there are `present`; their rank is 1.
  static __device__ __forceinline__ Cut Present(unsigned present) { return Cut{0, 0, present}; }
};

// Slots [from, to) of a sequence, in order, to their places in the kept list:
// those before lo and from hi on, and those between that the cut leaves. above,
// equal: what of its rank and above the slots between lo and `from` hold. The
// block's waves take a stretch each: they count, exchange the counts, and write.
template<class Rank>
__device__ __forceinline__ void WriteKept(std::uint32_t* kept, std::uint32_t from,
                                          std::uint32_t to, const EvictRange& range,
                                          const Cut& cut, unsigned above, unsigned equal,
                                          unsigned* s_above, unsigned* s_equal, Rank rank) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const std::uint32_t stretch =
      ((to - from + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
  const std::uint32_t begin = min(from + wave * stretch, to), end = min(begin + stretch, to);
  // Ranks of four runs of 64 slots, in flight together.
  constexpr int kRuns = 4;
  struct State {
    bool more, same;
  };
  const auto states = [&](std::uint32_t t0, State (&x)[kRuns]) {
    unsigned r[kRuns];
#pragma unroll
    for (int j = 0; j < kRuns; ++j)
      r[j] = rank(min(t0 + 64 * j + lane, end - 1));
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const std::uint32_t t = t0 + 64 * j + lane;
      const bool ranked = t < end && t >= range.lo && t < range.hi;
      x[j] = State{ranked && r[j] > cut.prefix, ranked && r[j] == cut.prefix};
    }
  };
  unsigned n_above = 0, n_equal = 0;
  for (std::uint32_t t0 = begin; t0 < end; t0 += 64 * kRuns) {
    State x[kRuns];
    states(t0, x);
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      n_above += __popcll(__ballot(x[j].more));
      n_equal += __popcll(__ballot(x[j].same));
    }
  }
  if (lane == 0) {
    s_above[wave] = n_above;
    s_equal[wave] = n_equal;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    above += s_above[w];
    equal += s_equal[w];
  }
  const unsigned long long before = (1ull << lane) - 1;
  for (std::uint32_t t0 = begin; t0 < end; t0 += 64 * kRuns) {
    State x[kRuns];
    states(t0, x);
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
      const std::uint32_t t = t0 + 64 * j + lane;
      const unsigned long long all_more = __ballot(x[j].more), all_same = __ballot(x[j].same);
      const unsigned my_above = above + __popcll(all_more & before);
      const unsigned my_equal = equal + __popcll(all_same & before);
      if (t < end && t < range.lo)
        kept[t] = t;
      else if (t < end && t >= range.hi)
        kept[range.lo + cut.ranked + (t - range.hi)] = t;
      else if (x[j].more || (x[j].same && my_equal < cut.need))
        kept[range.lo + my_above + min(my_equal, cut.need)] = t;
      above += __popcll(all_more);
      equal += __popcll(all_same);
    }
  }
}

// The slots that KV head g of sequence s keeps, in order, by one block. Where
// more slots are there than the budget, the rank of the last weight kept is
// found digit by digit over the slots between `sinks` and `recent`; else all that
// lie on a page are kept. What bounds it is the chain of its passes (32 lists of
// 2300 slots take 11 us, of which a launch is 3), not its 0.3 MB.
__launch_bounds__(kSelectThreads) __global__ void PagedSelectKernel(EvictArgs a) {
  extern __shared__ unsigned s_rank[];
  __shared__ unsigned s_bins[kBins], s_total[kSelectWaves], s_pick[2];
  __shared__ unsigned s_above[kSelectWaves], s_equal[kSelectWaves];
  const int g = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const EvictRange range(a, seq);
  const std::size_t list = std::size_t(seq) * a.kv_heads + g;
  std::uint32_t* kept = a.kept + list * a.budget;
  if (range.length <= a.budget) {
    const unsigned present = BlockTotal<kSelectWaves>(
        PresentShare(a.table, seq, range.lo, range.hi, kSelectThreads), s_total);
    if (a.counts && tid == 0)
      a.counts[list] = range.Count(present);
    if (present == range.hi - range.lo) {
      for (std::uint32_t i = tid; i < range.length; i += kSelectThreads)
        kept[i] = i;
      return;
    }
    WriteKept(kept, 0, range.length, range, Cut::Present(present), 0, 0, s_above, s_equal,
              [&](std::uint32_t t) { return a.table.Page(seq, t) < a.table.pages ? 1u : 0u; });
    return;
  }
  unsigned need = range.need, prefix = 0;  // fewer than there are
  if (need) {
    // Eight at a time: a page's number, then its weight, are a round trip each.
    for (std::uint32_t t0 = tid; t0 < range.length; t0 += 8 * kSelectThreads) {
      unsigned r[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        r[j] = ReadRank(a, seq, g, min(t0 + j * kSelectThreads, range.length - 1));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (t0 + j * kSelectThreads < range.length)
          s_rank[t0 + j * kSelectThreads] = r[j];
    }
    for (int d = 0; d < 3; ++d) {
      const Digit digit(d);
      s_bins[tid] = s_bins[tid + kSelectThreads] = 0;
      __syncthreads();
      for (std::uint32_t t = range.lo + tid; t < range.hi; t += kSelectThreads) {
        const unsigned r = s_rank[t];
        if ((r & digit.Before()) == prefix)
          atomicAdd(&s_bins[digit.Bin(r)], 1u);
      }
      __syncthreads();
      const uint2 pick = FindBin(s_bins[kBins - 1 - 2 * tid], s_bins[kBins - 2 - 2 * tid], need,
                                 s_total, s_pick);
      prefix |= pick.x << digit.low;
      need = pick.y;
    }
  }
  WriteKept(kept, 0, range.length, range, Cut::At(range.need, prefix, need), 0, 0, s_above,
            s_equal, [&](std::uint32_t t) { return s_rank[t]; });
}

// The same in slices of a sequence's slots, a block each, one launch a digit:
// every block adds up all slices' bins of the digit before, finds the same bin
// in them, and counts its own slots' next digit among those that are still in
// question; kDigit 3 writes the kept list. Each slice carries along how many
// slots of the slices before it rank above the threshold. Bound by the launches
// and what each reads again: 8 lists of 65,536 slots 5.9, 6.4, 6.5 and 8.6 us (in
// one block each, 153 in all).
template<int kDigit>
__launch_bounds__(kSelectThreads) __global__ void PagedSliceKernel(EvictArgs a, EvictSlices w) {
  __shared__ unsigned s_bins[kBins], s_total[kSelectWaves], s_pick[2];
  __shared__ unsigned s_above[kSelectWaves], s_equal[kSelectWaves];
  const int slice = blockIdx.x, g = blockIdx.y, seq = blockIdx.z, tid = threadIdx.x;
  const EvictRange range(a, seq);
  const std::uint32_t length = range.length, lo = range.lo, hi = range.hi;
  const std::uint32_t from = std::uint32_t(slice) * w.slice, to = min(from + w.slice, length);
  const std::size_t list = std::size_t(seq) * a.kv_heads + g,
                    lists = std::size_t(gridDim.z) * a.kv_heads;
  std::uint32_t* kept = a.kept + list * a.budget;
  if (length <= a.budget) {
    if constexpr (kDigit == 3) {
      const unsigned before = BlockTotal<kSelectWaves>(
          PresentShare(a.table, seq, lo, min(from, hi), kSelectThreads), s_total);
      const unsigned present = before + BlockTotal<kSelectWaves>(
          PresentShare(a.table, seq, max(lo, min(from, hi)), hi, kSelectThreads), s_total);
      if (slice == 0 && tid == 0)
        a.counts[list] = range.Count(present);
      if (from < to)
        WriteKept(kept, from, to, range, Cut::Present(present), before, 0, s_above, s_equal,
                  [&](std::uint32_t t) { return a.table.Page(seq, t) < a.table.pages ? 1u : 0u; });
    }
    return;
  }
  unsigned need = range.need, prefix = 0, above = 0, equal = 0;
  unsigned* ranks = w.ranks + list * w.slices * w.slice;
  if (kDigit > 0 && need) {
    const Digit last(kDigit - 1);
    if (kDigit > 1) {
      const uint2 s = w.state[(kDigit - 2) * lists + list];
      prefix = s.x;
      need = s.y;
    }
    // All slices' bins of the digit before; those of the slices before this
    // one apart.
    const unsigned* bins = w.bins + ((kDigit - 1) * lists + list) * w.slices * kBins;
    unsigned x[2] = {0, 0}, mine[2] = {0, 0};
    const int slices = int((length + w.slice - 1) / w.slice);
    constexpr int kBatch = 8;  // loads in flight
    for (int s0 = 0; s0 < slices; s0 += kBatch) {
      // Thread i's bins lie side by side: 2046 - 2 i, then 2047 - 2 i.
      uint2 y[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        y[j] = *reinterpret_cast<const uint2*>(bins + min(s0 + j, slices - 1) * kBins + kBins -
                                               2 - 2 * tid);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int s = s0 + j;
        x[0] += s < slices ? y[j].y : 0u;
        x[1] += s < slices ? y[j].x : 0u;
        mine[0] += s < slice ? y[j].y : 0u;
        mine[1] += s < slice ? y[j].x : 0u;
      }
    }
    const uint2 pick = FindBin(x[0], x[1], need, s_total, s_pick);
    const unsigned b0 = unsigned(kBins - 1 - 2 * tid);
    unsigned over = (b0 > pick.x ? mine[0] : 0u) + (b0 - 1 > pick.x ? mine[1] : 0u);
    unsigned same = (b0 == pick.x ? mine[0] : 0u) + (b0 - 1 == pick.x ? mine[1] : 0u);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      over += __shfl_xor(over, d);
      same += __shfl_xor(same, d);
    }
    if ((tid & 63) == 0) {
      s_above[tid >> 6] = over;
      s_equal[tid >> 6] = same;
    }
    __syncthreads();
    above = kDigit > 1 ? w.above[list * w.slices + slice] : 0u;
    for (int i = 0; i < kSelectWaves; ++i) {
      above += s_above[i];
      equal += s_equal[i];
    }
    __syncthreads();  // read before WriteKept counts there, and before it is carried on
    prefix |= pick.x << last.low;
    need = pick.y;
    if (kDigit < 3 && tid == 0) {
      w.above[list * w.slices + slice] = above;
      if (slice == 0)
        w.state[(kDigit - 1) * lists + list] = make_uint2(prefix, need);
    }
  }
  if constexpr (kDigit == 3) {
    const Cut cut = Cut::At(range.need, prefix, need);
    if (slice == 0 && tid == 0)
      a.counts[list] = range.Count(cut.ranked);
    if (from < to)
      WriteKept(kept, from, to, range, cut, above, equal, s_above, s_equal,
                [&](std::uint32_t t) { return ranks[t]; });
  } else {
    const Digit digit(kDigit);
    s_bins[tid] = s_bins[tid + kSelectThreads] = 0;
    __syncthreads();
    constexpr int kBatch = 4;
    for (std::uint32_t t0 = from + tid; t0 < to; t0 += kBatch * kSelectThreads) {
      unsigned r[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const std::uint32_t t = min(t0 + j * kSelectThreads, to - 1);
        r[j] = kDigit == 0 ? ReadRank(a, seq, g, t) : ranks[t];
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const std::uint32_t t = t0 + j * kSelectThreads;
        if (t >= to)
          continue;
        if (kDigit == 0)
          ranks[t] = r[j];
        if (t >= lo && t < hi && (r[j] & digit.Before()) == prefix)
          atomicAdd(&s_bins[digit.Bin(r[j])], 1u);
      }
    }
    __syncthreads();
    unsigned* bins = w.bins + ((kDigit * lists + list) * w.slices + slice) * kBins;
    bins[tid] = s_bins[tid];
    bins[tid + kSelectThreads] = s_bins[tid + kSelectThreads];
  }
}

// The kept slots' rows and weights to the new pages, D / 8 threads a slot, 16
// bytes each: bound by the copy (32 lists of 2048 slots, 67 MB both ways, 12 us:
// 5.6 TB/s out of the caches that hold part of it). How many there are is the
// same for every head; where no count was kept (lists of up to kOneBlock slots)
// each block adds up the table's pages while its rows are on their way.
template<int D>
__launch_bounds__(256) __global__ void PagedMoveKernel(EvictArgs a, std::uint32_t first) {
  constexpr int S = D / 8, kSlots = 256 / S;
  __shared__ unsigned s_wave[4];
  const int g = blockIdx.y, seq = blockIdx.z, seg = threadIdx.x % S;
  const EvictRange range(a, seq);
  const std::size_t list = std::size_t(seq) * a.kv_heads + g;
  const std::uint32_t most = min(range.length, a.budget);
  if (first + blockIdx.x * kSlots >= most)
    return;
  const std::uint32_t to = first + blockIdx.x * kSlots + threadIdx.x / S;
  const std::uint32_t from = a.kept[list * a.budget + min(to, most - 1)];
  const std::uint32_t page = a.table.Page(seq, from), new_page = a.new_table.Page(seq, to);
  // An entry that the list does not have reads some slot or page 0.
  const int page_slots = 1 << a.table.shift;
  const std::size_t src =
      (std::size_t(page < a.table.pages ? page : 0u) * a.kv_heads + g) * page_slots +
      (from & (page_slots - 1));
  const std::size_t dst =
      (std::size_t(new_page) * a.kv_heads + g) * page_slots + (to & (page_slots - 1));
  const uint4 k = reinterpret_cast<const uint4*>(a.k_pages)[src * S + seg];
  const uint4 v = reinterpret_cast<const uint4*>(a.v_pages)[src * S + seg];
  const float w = a.weight[src];
  std::uint32_t count;
  if (a.counts)
    count = a.counts[list];
  else
    count = range.Count(min(
        range.need,
        BlockTotal<4>(PresentShare(a.table, seq, range.lo, range.hi, 256), s_wave)));
  if (to >= count || page >= a.table.pages || new_page >= a.table.pages)
    return;
  reinterpret_cast<uint4*>(a.k_pages)[dst * S + seg] = k;
  reinterpret_cast<uint4*>(a.v_pages)[dst * S + seg] = v;
  if (seg == 0)
    a.weight[dst] = w;
}

// The slices of lists of up to max_length slots, and their workspace.
struct SlicePlan {
  std::uint32_t slice = 0, slices = 0;  // slices 0: one block a list
  std::size_t ranks = 0, bins = 0, state = 0, above = 0, counts = 0;  // bytes
  SlicePlan(std::size_t lists, std::uint32_t budget, std::uint32_t max_length) {
    if (max_length <= kOneBlock)
      return;
    counts = lists * sizeof(unsigned);
    if (max_length <= budget)
      return;
    slice = std::max(kSlice, (max_length + kMaxSlices - 1) / kMaxSlices);
    if (lists * ((max_length + slice - 1) / slice) > kCus)
      slice = std::max(slice, 2 * kSlice);
    slices = (max_length + slice - 1) / slice;
    ranks = lists * slices * slice * sizeof(unsigned);
    bins = 3 * lists * slices * kBins * sizeof(unsigned);
    state = 2 * lists * sizeof(uint2);
    above = lists * slices * sizeof(unsigned);
  }
  std::size_t Bytes() const { return bins + state + ranks + above + counts; }
};

}  // namespace
}  // namespace lfm3amd

using namespace lfm3amd;

extern "C" {

int lfm3_paged_heads(const lfm3_paged_cache* cache, const lfm3_paged_batch* batch,
                     const float* q, const float* k, const float* v, std::uint32_t ld,
                     const float* q_norm, const float* k_norm, const float* frequencies,
                     const float* factors, void* q_out, std::uint32_t ldq, std::uint32_t row_type,
                     std::uint32_t heads, float eps, void* stream) {
  int e = CheckPagedCache(cache);
  if (!e)
    e = CheckPagedBatch(batch);
  if (!e)
    e = CheckPagedRows(*cache, heads, row_type, q_out, ldq);
  if (!e)
    e = CheckPagedRows(*cache, heads, LFM3_TYPE_F32, q, ld);
  if (e)
    return e;
  if (!k || !v || !Aligned16(k) || !Aligned16(v) || !q_norm || !k_norm || !frequencies ||
      !batch->positions || ld < cache->kv_heads * cache->dim ||
      (q_out == q && (row_type != LFM3_TYPE_F32 || ldq != ld)))
    return Fail(LFM3_E_INVALID, "invalid LFM3 paged heads");
  if (!batch->rows)
    return LFM3_OK;
  HeadsArgs a{q, k, v, ld, q_norm, k_norm, frequencies, factors, q_out, ldq,
              static_cast<Half*>(cache->k), static_cast<Half*>(cache->v), cache->weight,
              PageTable{batch->tables, batch->table_stride, cache->pages, PageShift(cache->page)},
              batch->starts, batch->lengths, batch->positions, int(batch->seqs), int(heads),
              int(cache->kv_heads), eps, 0};
  const std::uint32_t rows = batch->rows, units = heads + 2 * cache->kv_heads;
  const auto s = static_cast<hipStream_t>(stream);
  const bool rows32 = row_type == LFM3_TYPE_F32, half = cache->type == LFM3_TYPE_F16;
  if (cache->dim == 128)
    half ? LaunchHeads<128, F16Pages>(a, rows, units, rows32, s)
         : LaunchHeads<128, Bf16Pages>(a, rows, units, rows32, s);
  else
    half ? LaunchHeads<64, F16Pages>(a, rows, units, rows32, s)
         : LaunchHeads<64, Bf16Pages>(a, rows, units, rows32, s);
  return HipStatus(hipGetLastError(), "LFM3 paged heads launch");
}

std::size_t lfm3_paged_evict_workspace_bytes(std::uint32_t seqs, std::uint32_t kv_heads,
                                             std::uint32_t budget, std::uint32_t max_length) {
  return SlicePlan(std::size_t(seqs) * kv_heads, budget, max_length).Bytes();
}

int lfm3_paged_evict(const lfm3_paged_cache* cache, const std::uint32_t* tables,
                     std::uint32_t table_stride, const std::uint32_t* lengths, std::uint32_t seqs,
                     std::uint32_t max_length, const std::uint32_t* new_tables,
                     std::uint32_t new_stride, std::uint32_t budget, std::uint32_t sinks,
                     std::uint32_t recent, std::uint32_t* kept, void* workspace,
                     std::size_t workspace_bytes, void* stream) {
  const int e = CheckPagedCache(cache);
  if (e)
    return e;
  if (!cache->weight || !tables || !table_stride || !lengths || !seqs || seqs > 65535 ||
      !new_tables || !kept || !budget || std::uint64_t(sinks) + recent > budget)
    return Fail(LFM3_E_INVALID, "invalid LFM3 paged eviction");
  if (std::size_t(new_stride) * cache->page < std::min(budget, max_length))
    return Fail(LFM3_E_INVALID, "LFM3 paged eviction: the new table is too short");
  if (max_length > kMaxLength)
    return Fail(LFM3_E_INVALID, "LFM3 paged eviction: too many slots");
  const SlicePlan plan(std::size_t(seqs) * cache->kv_heads, budget, max_length);
  if (workspace_bytes < plan.Bytes() || (plan.Bytes() && !workspace) || !Aligned16(workspace))
    return Fail(LFM3_E_INVALID, "LFM3 paged eviction workspace too small");
  const std::size_t reach = std::size_t(table_stride) * cache->page;
  max_length = std::uint32_t(std::min<std::size_t>(max_length, reach));
  if (!max_length)
    return LFM3_OK;
  const int shift = PageShift(cache->page);
  EvictArgs a{static_cast<Half*>(cache->k), static_cast<Half*>(cache->v), cache->weight,
              PageTable{tables, table_stride, cache->pages, shift},
              PageTable{new_tables, new_stride, cache->pages, shift}, lengths, max_length, budget,
              sinks, recent, kept, nullptr, int(cache->kv_heads)};
  const auto s = static_cast<hipStream_t>(stream);
  char* at = static_cast<char*>(workspace);
  if (plan.counts)
    a.counts = reinterpret_cast<unsigned*>(at + plan.Bytes() - plan.counts);
  if (plan.slices) {
    EvictSlices w;
    w.bins = reinterpret_cast<unsigned*>(at);
    w.state = reinterpret_cast<uint2*>(at + plan.bins);
    w.ranks = reinterpret_cast<unsigned*>(at + plan.bins + plan.state);
    w.above = reinterpret_cast<unsigned*>(at + plan.bins + plan.state + plan.ranks);
    w.slice = plan.slice;
    w.slices = plan.slices;
    const dim3 grid(plan.slices, cache->kv_heads, seqs);
    PagedSliceKernel<0><<<grid, kSelectThreads, 0, s>>>(a, w);
    PagedSliceKernel<1><<<grid, kSelectThreads, 0, s>>>(a, w);
    PagedSliceKernel<2><<<grid, kSelectThreads, 0, s>>>(a, w);
    PagedSliceKernel<3><<<grid, kSelectThreads, 0, s>>>(a, w);
  } else {
    const std::size_t ranks = std::min(max_length, kOneBlock) * sizeof(unsigned);
    const int status = HipStatus(
        hipFuncSetAttribute(reinterpret_cast<const void*>(PagedSelectKernel),
                            hipFuncAttributeMaxDynamicSharedMemorySize,
                            int(kOneBlock * sizeof(unsigned))),
        "LFM3 paged eviction shared memory");
    if (status)
      return status;
    PagedSelectKernel<<<dim3(cache->kv_heads, seqs), kSelectThreads, ranks, s>>>(a);
  }
  const std::uint32_t most = std::min(budget, max_length), slots = 256 * 8 / cache->dim;
  for (std::uint32_t first = 0; first < most; first += kMaxBlocks * slots) {
    const dim3 grid(std::min((most - first + slots - 1) / slots, kMaxBlocks), cache->kv_heads,
                    seqs);
    if (cache->dim == 128)
      PagedMoveKernel<128><<<grid, 256, 0, s>>>(a, first);
    else
      PagedMoveKernel<64><<<grid, 256, 0, s>>>(a, first);
  }
  return HipStatus(hipGetLastError(), "LFM3 paged eviction launch");
}

}  // extern "C"
