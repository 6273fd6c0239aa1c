// The attention weights that a batch's rows gave, summed into the paged cache's
// weights (lfm3_paged_weights) on gfx950 MFMA: weight[slot] += sum over rows
// and heads of exp(score - lse), the scores formed again as the attention forms
// them.
//
// S^T = K Q^T (rows are slots, columns (row, query head) pairs) leaves in lane L
// the slots 16 b + 4 (L / 16) + i of column L % 16; probabilities add up in that
// layout and meet over the columns at the end. Every slot has one owner, and
// nothing is added in an order that could change.
//
// One block of 8 waves a CU; each finds its work by scanning the batch's lengths
// itself (the host knows only their bound). Two shapes:
// * up to 16 columns (a decode row's group): all lists of slots (a sequence and
//   KV head each) in turns of 128 KB of K, shared out evenly and in order over
//   the blocks, whatever the lengths. K comes through each wave's own LDS stage,
//   requested as soon as the scores have read the last one. K is read once, and
//   that read is what bounds it: 24 rows over 8192 to 32,768 slots of 8 heads of
//   64 (0.5 GB) 113 us, 4.5 TB/s; 8 rows of up to 8192 slots 12.5 us, with the
//   launch and the scan.
// * more (a chunk): 64 slots or a few times that, K in registers as the A
//   operand; up to 8 waves share the columns of 64 slots and their sums add in
//   wave order. What bounds it is the exponentials and, where many waves share
//   columns, the reading of the queries (for FP32 rows also their split).
#include <algorithm>

#include "paged.hpp"

namespace lfm3amd {
namespace {

constexpr int kWaves = 8;
constexpr int kRuns = 4, kWideSlots = 16 * kRuns;  // slots a wave holds in registers
constexpr std::uint32_t kBlocks = 256;
// Decode rows' turns a block up to which it takes them from one list, and the
// blocks that these are reckoned for (every list rounds up).
constexpr int kFewTurns = 4, kNarrowUnits = 224;
constexpr std::uint64_t kMaxUnits = 0x7fffffff, kUnitSlots = std::uint64_t(kWaves) * kWideSlots;
constexpr std::size_t kNarrowLds = std::size_t(kWaves) * 16384;
constexpr float kLog2e = 1.44269504088896341f;

struct WeightsArgs {
  const void* q;
  std::size_t ldq;
  const float* lse;
  const Half* k_pages;
  float* weight;
  PageTable table;
  const std::uint32_t *starts, *lengths;
  int seqs, heads, kv_heads;
  std::uint32_t window, rows, max_length;
};

// A sequence's new rows and the slots [from, length) that they see, cut at
// max_length; rows 0: none.
struct Sequence {
  int first, rows, from, length;
  int before;  // the slot of the first row
};
__device__ __forceinline__ Sequence ReadSequence(const WeightsArgs& a, int s) {
  const std::uint32_t first = a.starts[s], end = a.starts[s + 1], length = a.lengths[s];
  Sequence x{0, 0, 0, 0, 0};
  if (end > first && end <= a.rows && length >= end - first && length <= kMaxLength) {
    x.first = int(first);
    x.rows = int(end - first);
    x.before = int(length) - x.rows;
    x.length = int(min(length, a.max_length));
    const int window = int(min(a.window, 0x7fffffffu));
    // From whole tiles of either shape on.
    x.from = window && x.before >= window ? (x.before + 1 - window) / 128 * 128 : 0;
    x.from = min(x.from, x.length);
  }
  return x;
}
// Waves that share a run of slots' columns, at most `most` of them.
__device__ __forceinline__ int Shares(int columns, int most) {
  return min(most, columns > 112 ? 8 : columns > 48 ? 4 : columns > 16 ? 2 : 1);
}
// Units of a sequence's list of slots for one KV head: turns of `size` slots
// (kNarrow: up to 16 columns), or what a block of waves holds at once where up
// to `size` of them share columns; 0 where the sequence is of the other shape.
template<bool kNarrow>
__device__ __forceinline__ int ListUnits(const Sequence& x, int group, int size) {
  const int columns = x.rows * group;
  if (!x.rows || (columns <= 16) != kNarrow)
    return 0;
  const int slots = kNarrow ? size : kWideSlots * kWaves / Shares(columns, size);
  return (x.length - x.from + slots - 1) / slots;
}

struct Unit {
  int seq, kv_head, index, count;  // unit `index` of the list's `count`
  Sequence rows;
};

// The batch's narrow turns, its wide units and the waves that may share columns
// in them: eight, unless those units would be more than blocks. Eight waves at
// one run of slots end it soonest; fewer hold more runs a block, and read the
// queries once for them. Every wave scans the sequences by itself, 64 a round
// trip.
struct Work {
  long long turns, wide;
  int shares;
};
__device__ __forceinline__ Work CountUnits(const WeightsArgs& a, int group, int turn, int lane) {
  long long turns = 0, wide[4] = {0, 0, 0, 0};
  for (int base = 0; base < a.seqs; base += 64) {
    Sequence x = ReadSequence(a, min(base + lane, a.seqs - 1));
    if (base + lane >= a.seqs)
      x.rows = 0;
    int n = ListUnits<true>(x, group, turn), m[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      m[k] = ListUnits<false>(x, group, 8 >> k);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      n += __shfl_xor(n, d);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        m[k] += __shfl_xor(m[k], d);
    }
    turns += (long long)(__builtin_amdgcn_readfirstlane(n)) * a.kv_heads;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      wide[k] += (long long)(__builtin_amdgcn_readfirstlane(m[k])) * a.kv_heads;
  }
  for (int k = 0; k < 3; ++k)
    if (wide[k] <= kBlocks)
      return Work{turns, wide[k], 8 >> k};
  return Work{turns, wide[3], 1};
}

// Unit `at` of the batch's units of a shape, lists in order of (sequence, KV
// head). Sums over 64 sequences fit 32 bits (kMaxUnits; a unit of a shape that is
// looked for here has 512 slots at least, or there are kBlocks of them at most).
template<bool kNarrow>
__device__ __forceinline__ Unit FindUnit(const WeightsArgs& a, long long at, int group, int size,
                                         int lane) {
  long long total = 0;
  for (int base = 0; base < a.seqs; base += 64) {
    Sequence x = ReadSequence(a, min(base + lane, a.seqs - 1));
    if (base + lane >= a.seqs)
      x.rows = 0;
    const int count = ListUnits<kNarrow>(x, group, size), mine = count * a.kv_heads;
    int upto = mine;  // units of this lane's sequence and those before it
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(upto, d);
      upto += lane >= d ? up : 0;
    }
    const unsigned long long after = __ballot(upto > at - total);
    if (after) {
      const int l = __ffsll(after) - 1;
      const auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      const int in = int(at - total) - pick(upto - mine), units = pick(count);
      return Unit{base + l, in / units, in % units, units,
                  Sequence{pick(x.first), pick(x.rows), pick(x.from), pick(x.length),
                           pick(x.before)}};
    }
    total += __builtin_amdgcn_readlane(upto, 63);
  }
  return Unit{0, 0, 0, 0, Sequence{0, 0, 0, 0, 0}};
}

// Four neighbouring weights, slots `slot` .. + 3 of a page.
__device__ __forceinline__ f4* Cells(const WeightsArgs& a, unsigned page, int g, int slot) {
  const int page_slots = 1 << a.table.shift;
  return reinterpret_cast<f4*>(a.weight +
                               (std::size_t(page) * a.kv_heads + g) * page_slots +
                               (slot & (page_slots - 1)));
}
// `old` with the sums of slots below `length` added.
__device__ __forceinline__ f4 Added(f4 old, f4 sum, int slot, int length) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    old[i] = slot + i < length ? old[i] + sum[i] : old[i];
  return old;
}

// Probabilities of scores s of a column: exp(s scale - lse), 0 where s is -inf.
__device__ __forceinline__ float Probability(float s, float scale, float minus_lse) {
  return __builtin_amdgcn_exp2f(fmaf(s, scale, minus_lse) * kLog2e);
}

// Up to 16 columns: slots [begin, end) of a list split over the waves. Here S = Q K^T, so
// that a lane's sums are of one slot: lane L holds columns 4 (L / 16) + i of slot
// 16 b + L % 16, adds its four, and the four lanes of a slot meet in two
// exchanges; lane L then owns slot 64 j + L of the tile.
template<int D, class T, bool kRows32>
__device__ __forceinline__ void NarrowSlots(const WeightsArgs& a, const Unit& unit, int begin,
                                            int end, int group, char* lds) {
  using Q = Query<D, T, kRows32>;
  using V8 = typename T::V8;
  constexpr int kKeys = 8192 / D, KB = kKeys / 16, kOwn = kKeys / 64;  // 16 KB of K a wave
  constexpr int kSteps = D / 32;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page_slots = 1 << a.table.shift;
  const Sequence& rows = unit.rows;
  // Uniform, but in part from vector divisions.
  const int g = __builtin_amdgcn_readfirstlane(unit.kv_head), seq = unit.seq;
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  char* tile = lds + wave * 16384;
  // The column's query first: its split does not wait for K.
  const int r = min(col / group, rows.rows - 1);
  const std::size_t row = unsigned(rows.first + r);
  const int head = g * group + col % group;
  Q raw;
  raw.Load(a.q, row * a.ldq + std::size_t(head) * D, lane);
  const float lse = a.lse[row * a.heads + head];
  int base = begin + wave * kKeys;
  constexpr int kStep = kWaves * kKeys;
  RunPages<KB> pages = FetchPages<KB>(a.table, seq, base, end);
  const HeadRows k_rows = HeadRows::Of<D>(a.k_pages, a.table, a.kv_heads, g);
  unsigned offset[StageShape<D>::kPerRun];
#pragma unroll
  for (int i = 0; i < StageShape<D>::kPerRun; ++i)
    offset[i] = StageShape<D>::LaneOffset(i, lane);
  StageOwnTile<D, kKeys>(a.table, k_rows, pages, base, end, offset, tile);
  // The lane's own weights: their places and what is summed so far.
  struct Cells {
    float* at[kOwn];
    float old[kOwn];
  };
  const auto read = [&](const RunPages<KB>& p, int from) {
    Cells x;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      unsigned page = ~0u;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        page = grp == k ? p.id[4 * j + k] : page;
      const int slot = from + 64 * j + lane;
      const bool mine = page < a.table.pages && slot < end;
      x.at[j] = mine ? a.weight + (std::size_t(page) * a.kv_heads + g) * page_slots +
                           (slot & (page_slots - 1))
                     : nullptr;
      x.old[j] = 0.0f;
      if (mine)
        x.old[j] = *x.at[j];
    }
    return x;
  };
  Cells cells = read(pages, base), done;  // of the tile at hand; of the one before, with its sums
#pragma unroll
  for (int j = 0; j < kOwn; ++j)
    done.at[j] = nullptr;
  const auto write = [&] {
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (done.at[j])
        *done.at[j] = done.old[j];
  };
  V8 q[Q::kParts][kSteps];
  float own_scale;
  raw.Split(q, own_scale);
  // What the lane needs of its four columns, from the lanes that loaded them.
  const bool live = col < rows.rows * group && lse != -INFINITY;
  const int seen = live ? rows.before + r : -1, window = int(min(a.window, 0x7fffffffu));
  float scale[4], minus_lse[4];
  int lo[4], hi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    scale[i] = __shfl(own_scale, 4 * grp + i);
    minus_lse[i] = __shfl(live ? -lse : 0.0f, 4 * grp + i);
    hi[i] = __shfl(seen, 4 * grp + i);
    lo[i] = window ? hi[i] + 1 - window : 0;
  }
  for (; base < end; base += kStep) {
    const RunPages<KB> next = FetchPages<KB>(a.table, seq, base + kStep, end);
    __builtin_amdgcn_s_waitcnt(WaitVm(0));
    asm volatile("" ::: "memory");
    f4 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      s[kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const int at = (16 * kb + col) * (D * 2) + ((4 * st + grp) ^ SlotSwizzle<D>(col)) * 16;
        const V8 k = *reinterpret_cast<const V8*>(tile + at);
#pragma unroll
        for (int p = 0; p < Q::kParts; ++p)
          s[kb] = T::Mfma(q[p][st], k, s[kb]);
      }
    }
    // The scores' reads are done before the stage is filled again. The sums of
    // the tile before go out ahead of that, so the wait above has them behind.
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    write();
    done = cells;
    cells = read(next, base + kStep);
    StageOwnTile<D, kKeys>(a.table, k_rows, next, base + kStep, end, offset, tile);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      float mine = 0.0f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int kb = 4 * j + k, t = base + 16 * kb + col;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = Probability(s[kb][i], scale[i], minus_lse[i]);
          sum += t >= lo[i] && t <= hi[i] ? p : 0.0f;
        }
        sum = SumXor32(SumXor16(sum));
        mine = grp == k ? sum : mine;
      }
      done.old[j] += mine;
    }
  }
  write();
  __builtin_amdgcn_s_waitcnt(WaitVm(0));  // loads past the stretch are still to land
  __syncthreads();  // what comes next may use the stages in another way
}

// The queries of a block's column tiles in LDS, two buffers in turn: a tile's
// parts as the product's operand takes them, then its columns' scales, negative
// lse and rows.
template<int D, class T, bool kRows32>
struct QueryStage {
  static constexpr int kParts = Query<D, T, kRows32>::kParts, kSteps = D / 32;
  static constexpr int kOperands = kParts * kSteps * 1024, kTile = kOperands + 256;
  // Column tiles a buffer: a wave's each, half as many where those of three
  // parts would not fit twice.
  static constexpr int kTiles = 2 * kWaves * kTile <= 144 * 1024 ? kWaves : kWaves / 2;
  static constexpr int kBytes = 2 * kTiles * kTile;
};

// More columns: K in registers, the columns shared by waves. Where four or
// eight share them (kAlone) each wave reads and splits the queries of its own
// column tiles. Where fewer do, every wave brings one of the next round's tiles
// into LDS, so that a tile is read and split once a block however many of its
// waves hold other slots: 300 rows of 16 heads over 24,000 slots 57 us, each for
// itself 79; with FP32 rows 89 and 147, over 12,000 60 and 81. (With eight, over
// 3000 slots, staging took 21 us against 20, with FP32 rows 41 against 28; with
// four, 200 rows of 32 heads of 2 KV heads and BF16 pages, 161 against 111:
// little is shared, and the rounds' barriers keep the waves in step.)
template<int D, class T, bool kRows32, bool kAlone>
__device__ __forceinline__ void WideUnit(const WeightsArgs& a, const Unit& unit, int group,
                                         int most, char* lds) {
  using V8 = typename T::V8;
  using Q = Query<D, T, kRows32>;
  using Stage = QueryStage<D, T, kRows32>;
  constexpr int kSteps = D / 32, KB = kRuns, kTiles = Stage::kTiles;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page_slots = 1 << a.table.shift;
  const int window = int(min(a.window, 0x7fffffffu));
  const int seq = unit.seq, g = unit.kv_head, rows = unit.rows.rows;
  const int length = unit.rows.length, before = unit.rows.before;
  const int columns = rows * group, tiles = (columns + 15) / 16, shares = Shares(columns, most);
  const int base =
      unit.rows.from + (unit.index * (kWaves / shares) + wave / shares) * kWideSlots;
  const RunPages<KB> pages = FetchPages<KB>(a.table, seq, base, length);
  // Column c of the sequence is row c / group, head c % group of the KV head; a
  // lane's columns are `stride` tiles apart, without a division each.
  const int stride = kAlone ? shares : kTiles;
  struct Column {
    Q raw;
    float lse;
    int row;  // among the sequence's
  };
  const unsigned c_first = unsigned(16 * (wave % stride) + col), c_step = unsigned(16 * stride);
  int load_row = int(c_first / unsigned(group)), load_head = int(c_first % unsigned(group));
  const int row_step = int(c_step / unsigned(group)), head_step = int(c_step % unsigned(group));
  const auto load = [&](Column& x) {
    const std::size_t row = unsigned(unit.rows.first + (load_row < rows ? load_row : 0));
    const int head = g * group + load_head;
    x.raw.Load(a.q, row * a.ldq + std::size_t(head) * D, lane);
    x.lse = a.lse[row * a.heads + head];
    x.row = load_row;
    load_row += row_step;
    load_head += head_step;
    const bool next = load_head >= group;
    load_head -= next ? group : 0;
    load_row += next ? 1 : 0;
  };
  // What the product needs of a column beside its query: the scale, -lse, the
  // last slot that its row sees, and whether it sees any (those behind the last
  // row see none, nor do rows whose attention saw none).
  const auto about = [&](const Column& x, float scale) {
    const bool live = x.row < rows && x.lse != -INFINITY;
    return f4{scale, live ? -x.lse : 0.0f, __int_as_float(before + x.row),
              __int_as_float(live ? 1 : 0)};
  };
  const auto store = [&](const Column& x, int buffer) {
    if (wave >= kTiles)
      return;
    V8 q[Q::kParts][kSteps];
    float scale;
    x.raw.Split(q, scale);
    char* at = lds + (buffer * kTiles + wave) * Stage::kTile;
#pragma unroll
    for (int p = 0; p < Q::kParts; ++p)
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        *reinterpret_cast<V8*>(at + (p * kSteps + s) * 1024 + lane * 16) = q[p][s];
    if (grp == 0)
      *reinterpret_cast<f4*>(at + Stage::kOperands + col * 16) = about(x, scale);
  };
  // The next tiles' queries are on their way behind the one at hand, in buffers
  // that take turns (a copy of one would wait for its loads). Alone, FP32 rows
  // hide one behind the split of the other; 16-bit rows take two.
  constexpr int kRing = kAlone && !kRows32 ? 3 : 2;
  Column ring[kRing];
#pragma unroll
  for (int i = 0; i < (kAlone ? kRing - 1 : 2); ++i)
    load(ring[i]);
  V8 k[KB][kSteps];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int t = base + 16 * kb;
    const bool there = pages.id[kb] < a.table.pages;
    const Half* rows_of =
        a.k_pages + (std::size_t(there ? pages.id[kb] : 0u) * a.kv_heads + g) * page_slots * D;
    const BufferResource res = MakeBuffer(rows_of, unsigned(page_slots * D * 2));
    const unsigned offset = unsigned(((t + col) & (page_slots - 1)) * D * 2 + 16 * grp);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      k[kb][s] = __builtin_bit_cast(
          V8, LoadB128(res, there && t + col < length ? offset + 64 * s : kOutOfRange));
  }
  // Lane 4 kb + grp of the run's first wave owns slots 16 kb + 4 grp .. + 3.
  const int own_slot = 4 * lane;
  unsigned own_page = ~0u;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
    own_page = (lane >> 2) == kb ? pages.id[kb] : own_page;
  const bool owner =
      wave % shares == 0 && own_page < a.table.pages && base + own_slot < length;
  f4 old = f4{0.0f, 0.0f, 0.0f, 0.0f};
  if (owner)
    old = *Cells(a, own_page, g, base + own_slot);
  if constexpr (!kAlone) {
    store(ring[0], 0);
    load(ring[0]);
  }

  f4 sum[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
    sum[kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  // A tile's queries against the wave's slots; operand(p, s): of part p, step s.
  const auto step = [&](const f4& column, const auto& operand) {
    const float scale = column[0], minus_lse = column[1];
    const int own = __float_as_int(column[2]), hi = __float_as_int(column[3]) ? own : -1;
    const int lo = window ? own + 1 - window : 0;
    // The tile's rows (those past the last one see nothing): what they see
    // between them, and each of them.
    const int r0 = __builtin_amdgcn_readfirstlane(own);
    const int r1 = __builtin_amdgcn_readlane(own, 15);
    if (base > r1 || (window && base + kWideSlots - 1 <= r0 - window))
      return;
    const bool open = base + kWideSlots - 1 <= r0 && (!window || base > r1 - window) &&
                      !__ballot(hi < 0);
    f4 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      s[kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    // The runs' chains side by side.
#pragma unroll
    for (int p = 0; p < Q::kParts; ++p)
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const V8 q = operand(p, st);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          s[kb] = T::Mfma(k[kb][st], q, s[kb]);
      }
    if (!open) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int t = base + 16 * kb + 4 * grp + i;
          s[kb][i] = t >= lo && t <= hi ? s[kb][i] : -INFINITY;
        }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sum[kb][i] += Probability(s[kb][i], scale, minus_lse);
  };
  if constexpr (kAlone) {
    const auto turn = [&](const Column& now, Column& later) {
      load(later);
      V8 q[Q::kParts][kSteps];
      float scale;
      now.raw.Split(q, scale);
      step(about(now, scale), [&](int p, int s) { return q[p][s]; });
    };
    // K has to be there before the loop: waited for inside it, by count, each
    // turn would wait for the queries that it has just asked for.
    __builtin_amdgcn_s_waitcnt(WaitVm(0));
    int tile = wave % shares;
    const int stop = base < length ? tiles : 0;
    // The buffers take turns by position, and the only way on is out: with a path
    // that skips a turn, a load would wait for what that path has pending.
    if (tile < stop)
      for (;;) {
        turn(ring[0], ring[kRing - 1]);
        if ((tile += stride) >= stop)
          break;
        turn(ring[1], ring[0]);
        if ((tile += stride) >= stop)
          break;
        if constexpr (kRing == 3) {
          turn(ring[2], ring[1]);
          if ((tile += stride) >= stop)
            break;
        }
      }
  } else {
    const bool busy = base < length;
    int first = 0;  // the round's first tile
    // The round's tiles, from `buffer`; then the next round's queries, from `x`,
    // into the other one.
    const auto round = [&](int buffer, Column& x) {
      // The round's queries are there, and those before them read.
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
      BlockBarrier();
      const int end = busy ? min(kTiles, tiles - first) : 0;
      for (int tile = wave % shares; tile < end; tile += shares) {
        const char* at = lds + (buffer * kTiles + tile) * Stage::kTile;
        step(*reinterpret_cast<const f4*>(at + Stage::kOperands + col * 16), [&](int p, int s) {
          return *reinterpret_cast<const V8*>(at + (p * kSteps + s) * 1024 + lane * 16);
        });
      }
      first += kTiles;
      if (first < tiles)
        store(x, buffer ^ 1);
      load(x);
    };
    while (first < tiles) {
      round(0, ring[1]);
      if (first >= tiles)
        break;
      round(1, ring[0]);
    }
  }
  __syncthreads();  // the sums go where queries were
  const auto s_sum = reinterpret_cast<f4(*)[4 * kRuns]>(lds);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    f4 total;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      total[i] = GroupSum16(sum[kb][i]);
    if (col == 0)
      s_sum[wave][4 * kb + grp] = total;
  }
  __syncthreads();
  if (owner) {
    f4 total = s_sum[wave][lane];
    for (int w = 1; w < shares; ++w)
      total += s_sum[wave + w][lane];
    *Cells(a, own_page, g, base + own_slot) = Added(old, total, base + own_slot, length);
  }
  __syncthreads();  // the sums are read before the next slots' are written
}

template<int D, class T, bool kRows32>
__launch_bounds__(64 * kWaves, 2) __global__ void PagedWeightsKernel(WeightsArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int group = a.heads / a.kv_heads, lane = threadIdx.x & 63;
  constexpr int kTurn = kWaves * 8192 / D;  // slots that the waves' stages hold
  static_assert(kTurn >= int(kUnitSlots), "the host's bound of the units");
  const Work work = CountUnits(a, group, kTurn, lane);
  const long long turns = work.turns;
  const int few = int(min((turns + kNarrowUnits - 1) / kNarrowUnits, 1ll << 20));
  if (few <= kFewTurns) {
    // Few turns a block: each takes that many of one list, so that none starts
    // on a second list (8 sequences of 128 to 8192 slots: 14.7 us, 19.1 shared
    // out evenly; the 24 of 8192 to 32768: 163 us, 114 evenly).
    for (long long at = blockIdx.x; at < turns; at += gridDim.x) {
      const Unit unit = FindUnit<true>(a, at, group, few * kTurn, lane);
      if (!unit.count)
        break;
      const int begin = unit.rows.from + unit.index * few * kTurn;
      NarrowSlots<D, T, kRows32>(a, unit, begin, min(begin + few * kTurn, unit.rows.length),
                                 group, lds);
    }
  } else {
    const long long last = turns * (blockIdx.x + 1) / gridDim.x;
    for (long long at = turns * blockIdx.x / gridDim.x; at < last;) {
      const Unit unit = FindUnit<true>(a, at, group, kTurn, lane);
      if (!unit.count)
        break;
      const int n = int(min(last - at, (long long)(unit.count - unit.index)));
      const int begin = unit.rows.from + unit.index * kTurn;
      NarrowSlots<D, T, kRows32>(a, unit, begin, min(begin + n * kTurn, unit.rows.length), group,
                                 lds);
      at += n;
    }
  }
  for (long long at = blockIdx.x; at < work.wide; at += gridDim.x) {
    const Unit unit = FindUnit<false>(a, at, group, work.shares, lane);
    if (!unit.count)
      break;
    if (Shares(unit.rows.rows * group, work.shares) > 2)
      WideUnit<D, T, kRows32, true>(a, unit, group, work.shares, lds);
    else
      WideUnit<D, T, kRows32, false>(a, unit, group, work.shares, lds);
  }
}

template<int D, class T, bool kRows32>
int LaunchKernel(const WeightsArgs& a, hipStream_t s) {
  const auto kernel = PagedWeightsKernel<D, T, kRows32>;
  constexpr std::size_t kLds =
      std::max<std::size_t>(kNarrowLds, QueryStage<D, T, kRows32>::kBytes);
  const int e = HipStatus(
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, int(kLds)),
      "LFM3 paged weights shared memory");
  if (e)
    return e;
  kernel<<<kBlocks, 64 * kWaves, kLds, s>>>(a);
  return HipStatus(hipGetLastError(), "LFM3 paged weights launch");
}
template<int D, class T>
int Launch(const WeightsArgs& a, bool rows32, hipStream_t s) {
  return rows32 ? LaunchKernel<D, T, true>(a, s) : LaunchKernel<D, T, false>(a, s);
}

}  // namespace
}  // namespace lfm3amd

using namespace lfm3amd;

extern "C" int lfm3_paged_weights(const lfm3_paged_cache* cache, const lfm3_paged_batch* batch,
                                  const void* q, std::uint32_t ldq, std::uint32_t row_type,
                                  const float* lse, std::uint32_t heads, std::uint32_t window,
                                  std::uint32_t max_length, void* stream) {
  int e = CheckPagedCache(cache);
  if (!e)
    e = CheckPagedBatch(batch);
  if (!e)
    e = CheckPagedRows(*cache, heads, row_type, q, ldq);
  if (e)
    return e;
  if (!cache->weight || !lse)
    return Fail(LFM3_E_INVALID, "LFM3 paged weights need the cache's weights and the rows' lse");
  const std::size_t reach = std::size_t(batch->table_stride) * cache->page;
  max_length = std::uint32_t(std::min<std::size_t>(std::min<std::size_t>(max_length, reach),
                                                   kMaxLength));
  if (!batch->rows || !max_length)
    return LFM3_OK;
  if (std::uint64_t(std::min(batch->seqs, 64u)) * cache->kv_heads *
          ((max_length + kUnitSlots - 1) / kUnitSlots) > kMaxUnits)
    return Fail(LFM3_E_INVALID, "LFM3 paged weights: too many slots");
  const WeightsArgs a{q, ldq, lse, static_cast<const Half*>(cache->k), cache->weight,
                      PageTable{batch->tables, batch->table_stride, cache->pages,
                                PageShift(cache->page)},
                      batch->starts, batch->lengths, int(batch->seqs), int(heads),
                      int(cache->kv_heads), window, batch->rows, max_length};
  const auto s = static_cast<hipStream_t>(stream);
  const bool rows32 = row_type == LFM3_TYPE_F32, half = cache->type == LFM3_TYPE_F16;
  if (cache->dim == 128)
    return half ? Launch<128, F16Pages>(a, rows32, s) : Launch<128, Bf16Pages>(a, rows32, s);
  return half ? Launch<64, F16Pages>(a, rows32, s) : Launch<64, Bf16Pages>(a, rows32, s);
}
