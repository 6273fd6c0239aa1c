// Attention of packed rows over the paged cache on gfx950 MFMA: chunks of
// prompts and single tokens, of several sequences, in one launch.
//
// A block of 8 waves takes one item of the plan: a row tile of a sequence, one
// KV head and a span of its slots. The tile's columns are its (row, query
// head of the group) pairs. Every wave forms S^T = K Q^T (rows are slots,
// columns the pairs), the base-2 online softmax of its columns, and O^T += V^T
// P^T, both on v_mfma_f32_16x16x32. The accumulator of S^T leaves in lane L
// the slots 16 b + 4 (L / 16) + i of column L % 16, and the products over
// slots take them from there: the order of a product's 32 slots is free as
// long as both operands agree, so V^T's operand is read in that order
// (ds_read_b64_tr_b16 hands a lane four slots of one dimension) and
// probabilities never cross lanes.
//
// K and V arrive by direct-to-LDS buffer loads, each wave instruction within
// one run of 16 slots and so on one page: its resource is the run's rows up to
// the span's end, formed from 64-bit addresses in scalar registers (a pool may
// pass 4 GiB), so that lanes' offsets never change; slots past the end, and runs
// on no page, read as zeros. A row's 16-byte segments lie XORed with the slot so
// that operand reads meet distinct banks.
//
// Two shapes of the same work:
// * up to 16 columns (a decode row's group): the waves split the span, each
//   through its own LDS stage without a block barrier. The next K tile is
//   requested when the scores have read the last one and the next V tile when
//   the outputs have, so each is in flight while the other is used, 128 KB a
//   CU in all; the waves meet in LDS at the end. Bound by the read of K and V:
//   24 rows over 8192 to 32,768 slots of 8 heads of 64 (1.0 GB) 180 us, 5.7 TB/s
//   of the 6.1 that a bare read reaches. 8 rows of up to 8192 slots (75 MB) are
//   14 us, a third of it the launch, the pages' numbers and the last joins.
// * more (a chunk): the waves split the columns, 16 or 32 each, over shared
//   tiles of 64 slots in a three-stage ring with one barrier a tile. A stage is
//   one of K and V; three leave two tiles' loads in flight behind the one at
//   hand. Bound by the chain of products, softmax and products of a wave, which
//   two waves a SIMD overlap in part: 512 F16 rows of 16 heads of 128 over 24,576
//   slots (104 GFLOP) 114 us without the merge, 0.91 PFLOP/s, where the matrix
//   cores' loop alone reaches 2.3. (That is call after call; the first 10 ms after
//   an idle card, before the clock has settled, 134 to 145 us.)
//
// Split tiles leave a record a (row, head): the unnormalized output, the
// maximum, the sum and the scale; PagedMergeKernel adds a row's records in
// span order.
//
// FP32 rows: query rows enter in parts (Query), and a probability in as many of
// its type. Rows of the pages' type enter whole; a probability rounds to that
// type once. F16 probabilities, of either rows, are taken times 2^15: those down
// to 2^-29 of the column's largest are normal values (rounded by 2^-11 of
// themselves, no more than the output will be; two parts by 2^-22 down to 2^-18),
// and none is off by more than 2^-40 of the largest. Unscaled, a long tail of
// slots e^-17 below a first slot without a value lost a third of the output. The
// sum adds the FP32 values in both, for the rows' lse.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "paged.hpp"

namespace lfm3amd {
namespace {

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr std::uint32_t kNarrowColumns = 16, kHalfColumns = 16 * kWaves;
constexpr std::uint32_t kTileColumns = 2 * kHalfColumns;  // of a full row tile
constexpr int kStages = 3, kWideKeys = 64;
constexpr std::uint32_t kMaxParts = 64;

struct AttentionArgs {
  const void* q;
  std::size_t ldq;
  const float* gate;
  std::size_t ldg;
  void* out;
  std::size_t ldo;
  float* lse;
  const Half *k_pages, *v_pages;
  PageTable table;
  const lfm3_paged_item* items;
  float* records;
  std::uint32_t max_records, seqs, rows, window;
  int heads, kv_heads;
};

// Floats of a record: the output, the maximum, the sum, the scale.
constexpr int RecordFloats(int dim) { return dim + 4; }
constexpr std::size_t RecordBytes(std::size_t heads, std::uint32_t dim) {
  return heads * RecordFloats(int(dim)) * sizeof(float);
}

// An item whose parts all lie inside the batch, the table and the workspace.
__device__ __forceinline__ bool Sound(const AttentionArgs& a, const lfm3_paged_item& it,
                                      int group) {
  return it.seq < a.seqs && it.row <= a.rows && it.rows <= a.rows - it.row && it.rows &&
         it.rows <= kTileColumns / unsigned(group) && it.part < it.parts &&
         it.slot <= kMaxLength && it.key_begin < it.key_end && it.key_end <= kMaxLength &&
         it.kv_head < unsigned(a.kv_heads) &&
         (it.parts == 1 ||
          (it.record <= a.max_records && it.rows <= a.max_records - it.record));
}

__device__ __forceinline__ lfm3_paged_item UniformItem(const lfm3_paged_item* items) {
  typedef const __attribute__((address_space(4))) lfm3_paged_item Constant;
  Constant& it = ((Constant*)items)[blockIdx.x];
  return lfm3_paged_item{it.seq,     it.row,  it.rows,  it.slot,   it.key_begin,
                         it.key_end, it.part, it.parts, it.record, it.kv_head, {0, 0}};
}

// The softmax state of CT tiles of 16 columns in one wave.
template<int D, class T, bool kRows32, int CT>
struct Columns {
  using V8 = typename T::V8;
  static constexpr bool kHalf = T::kType == LFM3_TYPE_F16;
  static constexpr int kParts = Query<D, T, kRows32>::kParts;
  static constexpr int kSteps = D / 32, kDims = D / 16;
  static constexpr float kPScale = kHalf ? 32768.0f : 1.0f;  // of probabilities and outputs
  static constexpr float kPLog2 = kHalf ? 15.0f : 0.0f;

  V8 q[CT][kParts][kSteps];
  float scale[CT];  // of raw scores, in units of the natural logarithm
  f4 acc[CT][kDims];
  float m[CT], l[CT];  // l: the lane's own slots (16-bit rows: of scaled probabilities)
  int lo[CT], hi[CT];  // slots that the column sees in the span, inclusive

  // The wave's columns begin at column `first` of the item.
  __device__ __forceinline__ void Load(const AttentionArgs& a, const lfm3_paged_item& it,
                                       int group, int first, int lane) {
    const int col = lane & 15;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const unsigned c = unsigned(first + 16 * ct + col), r = c / unsigned(group);
      const bool live = r < it.rows;
      const std::size_t row = it.row + (live ? r : 0u);
      const int head = int(it.kv_head) * group + int(live ? c % unsigned(group) : 0u);
      const int own = int(it.slot + r);
      const int oldest = a.window && unsigned(own) >= a.window ? own + 1 - int(a.window) : 0;
      lo[ct] = live ? max(oldest, int(it.key_begin)) : 0x7fffffff;
      hi[ct] = live ? min(own, int(it.key_end) - 1) : -1;
      m[ct] = -INFINITY;
      l[ct] = 0.0f;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
        acc[ct][d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      Query<D, T, kRows32> query;
      query.Load(a.q, row * a.ldq + std::size_t(head) * D, lane);
      query.Split(q[ct], scale[ct]);
    }
  }

  template<int KB>
  __device__ __forceinline__ void Scores(const char* tile, int lane, f4 (&s)[CT][KB]) const {
    TileScores<D, T>(tile, lane, q, s);
  }

  // Scores of slots base + ... to the probabilities' operands. kOpen: every
  // column sees every slot; holes: bit kb set where run kb is on no page.
  template<int KB, bool kOpen>
  __device__ __forceinline__ void Softmax(f4 (&s)[CT][KB], int base, unsigned holes, int lane,
                                          V8 (&p)[CT][kParts][KB / 2]) {
    const int grp = lane >> 4;
    constexpr float kLog2e = 1.44269504088896341f;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if constexpr (!kOpen) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int t = base + 16 * kb + 4 * grp + i;
            const bool seen = t >= lo[ct] && t <= hi[ct] && !(holes >> kb & 1u);
            s[ct][kb][i] = seen ? s[ct][kb][i] : -INFINITY;
          }
      }
      float top = s[ct][0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = fmaxf(top, s[ct][kb][i]);
      const float next = fmaxf(m[ct], MaxXor32(MaxXor16(top)));
      const float shift = next == -INFINITY ? 0.0f : next, c = scale[ct] * kLog2e;
      const float alpha = __builtin_amdgcn_exp2f((m[ct] - shift) * c);
      m[ct] = next;
      // 16-bit rows: one multiply-add a score, s c - shift c, whose constant rounds
      // by as much as a score itself does. Where that could pass 2^-4 (the largest
      // probability would be 2^it, past F16's range or nothing at scores of 10^8),
      // the shift is taken off first, as FP32 rows always do. The probability's
      // scale comes by way of the exponent too; Sum() takes it out again.
      float base2 = fmaf(-shift, c, kPLog2);
      if constexpr (!kRows32) {
        if (__ballot(fabsf(base2) >= 0x1p20f)) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
            s[ct][kb] -= shift;
          base2 = kPLog2;
        }
      }
      typedef float f2 __attribute__((ext_vector_type(2)));
      typedef _Float16 e2 __attribute__((ext_vector_type(2)));
      typedef __bf16 b2 __attribute__((ext_vector_type(2)));
      using V2 = std::conditional_t<kHalf, e2, b2>;
      unsigned w[kParts][KB][2];
      float local[2] = {0.0f, 0.0f};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float s0 = s[ct][kb][2 * j], s1 = s[ct][kb][2 * j + 1];
          if constexpr (kRows32) {
            // The difference before the scale: what rounds is its own size.
            const float p0 = __builtin_amdgcn_exp2f((s0 - shift) * c);
            const float p1 = __builtin_amdgcn_exp2f((s1 - shift) * c);
            local[0] += p0;
            local[1] += p1;
            f2 rest = {p0 * kPScale, p1 * kPScale};
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const V2 r = __builtin_convertvector(rest, V2);
              w[part][kb][j] = __builtin_bit_cast(unsigned, r);
              rest = f2{rest[0] - float(r[0]), rest[1] - float(r[1])};
            }
          } else {
            const f2 e = {__builtin_amdgcn_exp2f(fmaf(s0, c, base2)),
                          __builtin_amdgcn_exp2f(fmaf(s1, c, base2))};
            local[0] += e[0];
            local[1] += e[1];
            w[0][kb][j] = __builtin_bit_cast(unsigned, __builtin_convertvector(e, V2));
          }
        }
      l[ct] = l[ct] * alpha + (local[0] + local[1]);
      // 2^0 is exactly 1: where no column's maximum moved nothing is rescaled.
      if (__ballot(alpha != 1.0f)) {
#pragma unroll
        for (int d = 0; d < kDims; ++d)
          acc[ct][d] *= alpha;
      }
#pragma unroll
      for (int c2 = 0; c2 < KB / 2; ++c2)
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
          const unsigned x[4] = {w[part][2 * c2][0], w[part][2 * c2][1], w[part][2 * c2 + 1][0],
                                 w[part][2 * c2 + 1][1]};
          p[ct][part][c2] = Pack4<V8>(x);
        }
    }
  }

  // A column's sum of probabilities, in all its lanes.
  __device__ __forceinline__ float Sum(int ct) const {
    return SumXor32(SumXor16(l[ct])) * (kRows32 ? 1.0f : 1.0f / kPScale);
  }

  // V^T operand: dimension 16 d + L % 16, slots 32 c2 + 4 (L / 16) + 0..3 and
  // those 16 later.
  static __device__ __forceinline__ V8 Values(const char* tile, int lane, int c2, int d) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 Lds4;
    typedef short s8 __attribute__((ext_vector_type(8)));
    const int low = 4 * (lane >> 4) + ((lane & 15) >> 2);  // the slot in its run
    const int at = (32 * c2 + low) * (D * 2) +
                   ((2 * d + ((lane & 3) >> 1)) ^ SlotSwizzle<D>(low)) * 16 + (lane & 1) * 8;
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)(tile + at));
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4*)(tile + at + 16 * D * 2));
    return __builtin_bit_cast(V8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // O^T += V^T P^T.
  template<int KB>
  __device__ __forceinline__ void Outputs(const char* tile, int lane,
                                          const V8 (&p)[CT][kParts][KB / 2]) {
    if constexpr (CT == 2) {
      // Products enough to each operand: the order is left to the compiler.
#pragma unroll
      for (int c2 = 0; c2 < KB / 2; ++c2)
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          const V8 v = Values(tile, lane, c2, d);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
#pragma unroll
            for (int part = 0; part < kParts; ++part)
              acc[ct][d] = T::Mfma(v, p[ct][part][c2], acc[ct][d]);
        }
    } else {
      // kGroup operands are read while the kGroup before them are multiplied:
      // 512 FP32 rows of 16 heads of 128 over 24,576 F16 slots, one column tile
      // a wave, 217 us, 224 with the order left to the compiler. (With CT 2, 32
      // heads of 64, it is 234 and 228 us.)
      constexpr int kGroup = 4, kGroups = KB / 2 * kDims / kGroup;
      V8 v[2][kGroup];
      const auto read = [&](int n) {
#pragma unroll
        for (int j = 0; j < kGroup; ++j)
          v[n & 1][j] = Values(tile, lane, (n * kGroup + j) / kDims, (n * kGroup + j) % kDims);
      };
      read(0);
#pragma unroll
      for (int n = 0; n < kGroups; ++n) {
        if (n + 1 < kGroups)
          read(n + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int part = 0; part < kParts; ++part)
#pragma unroll
          for (int j = 0; j < kGroup; ++j) {
            const int c2 = (n * kGroup + j) / kDims, d = (n * kGroup + j) % kDims;
            acc[0][d] = T::Mfma(v[n & 1][j], p[0][part][c2], acc[0][d]);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }

  // Whether the tile's V holds an infinity or NaN.
  template<int KB>
  static __device__ __forceinline__ bool Poisoned(const char* tile, int lane) {
    constexpr unsigned kTop = kHalf ? 0x7c007c00u : 0x7f807f80u;
    constexpr unsigned kLow = kHalf ? 0x04000400u : 0x00800080u;
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < 16 * KB * D / 512; ++i) {
      const uint4 x = *reinterpret_cast<const uint4*>(tile + (i * 64 + lane) * 16);
      // An exponent of all ones carries into the sign's place.
      carry |= (((x.x & kTop) + kLow) | ((x.y & kTop) + kLow) | ((x.z & kTop) + kLow) |
                ((x.w & kTop) + kLow)) & 0x80008000u;
    }
    return __ballot(carry != 0) != 0;
  }

  // O^T += V^T P^T where some columns do not see some slots and V holds
  // infinities or NaN: 0 times those would reach columns that do not see
  // them. The finite values go as above; the others are added to the columns
  // that see their slot.
  template<int KB>
  __device__ __forceinline__ void OutputsApart(const char* tile, int lane, int base,
                                               const V8 (&p)[CT][kParts][KB / 2]) {
    constexpr unsigned kExp = kHalf ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int c2 = 0; c2 < KB / 2; ++c2)
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        typedef unsigned u4 __attribute__((ext_vector_type(4)));
        const u4 v = __builtin_bit_cast(u4, Values(tile, lane, c2, d));
        unsigned finite[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          finite[j] = ((v[j] & kExp) == kExp ? 0u : v[j] & 0xffffu) |
                      ((v[j] >> 16 & kExp) == kExp ? 0u : v[j] & 0xffff0000u);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int part = 0; part < kParts; ++part)
            acc[ct][d] = T::Mfma(Pack4<V8>(finite), p[ct][part][c2], acc[ct][d]);
        __builtin_amdgcn_sched_barrier(0);  // one operand at a time: registers
      }
#pragma unroll 1
    for (int key = 0; key < 16 * KB; ++key) {
      const char* at = tile + key * (D * 2);
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        // Dimensions 16 d + 4 (L / 16) + 0..3, the lane's own outputs.
        const int seg = 2 * d + (lane >> 5);
        const uint2 v = *reinterpret_cast<const uint2*>(
            at + (seg ^ SlotSwizzle<D>(key & 15)) * 16 + (lane >> 4 & 1) * 8);
        const unsigned x[4] = {v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16};
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bool seen = base + key >= lo[ct] && base + key <= hi[ct];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[ct][d][i] += seen && (x[i] & kExp) == kExp ? T::Load(x[i]) : 0.0f;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// What rows r0 .. r1 of the item (as slots) see in its span: between them
// [reach_lo, reach_hi], each of them all of [whole_lo, whole_hi].
struct Sight {
  int reach_lo, reach_hi, whole_lo, whole_hi;
  __device__ __forceinline__ Sight(const lfm3_paged_item& it, std::uint32_t window, int r0,
                                   int r1) {
    const int w = int(min(window, 0x7fffffffu)), begin = int(it.key_begin);
    // Uniform, but by way of vector divisions.
    const auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    reach_lo = scalar(max(begin, w && r0 >= w ? r0 + 1 - w : 0));
    whole_lo = scalar(max(begin, w && r1 >= w ? r1 + 1 - w : 0));
    reach_hi = scalar(min(r1, int(it.key_end) - 1));
    whole_hi = scalar(min(r0, int(it.key_end) - 1));
  }
};

// A (row, head)'s gate, before its sigmoid; infinity, whose sigmoid is 1,
// without gates.
__device__ __forceinline__ float Gate(const AttentionArgs& a, std::size_t row, int head) {
  return a.gate ? a.gate[row * a.ldg + head] : INFINITY;
}
// Four neighbouring outputs of a (row, head), normalized and gated, or the
// record's four. l 0: the row sees nothing.
template<int D, class T, bool kRows32, float kPScale>
__device__ __forceinline__ void StoreOutputs(const AttentionArgs& a, std::size_t row, int head,
                                             int d, const float (&x)[4], float l, float raw) {
  const float gate = 1.0f + expf(-raw);
  const float inv = l != 0.0f ? 1.0f / (l * kPScale) : 0.0f;
  const std::size_t at = row * a.ldo + std::size_t(head) * D + d;
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    y[i] = x[i] * inv / gate;
  if constexpr (kRows32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) =
        make_float4(y[0], y[1], y[2], y[3]);
  } else {
    const unsigned u = T::Round(y[0]) | unsigned(T::Round(y[1])) << 16;
    const unsigned v = T::Round(y[2]) | unsigned(T::Round(y[3])) << 16;
    *reinterpret_cast<uint2*>(static_cast<Half*>(a.out) + at) = make_uint2(u, v);
  }
}
template<int D>
__device__ __forceinline__ float* Record(const AttentionArgs& a, const lfm3_paged_item& it,
                                         std::size_t row, int head) {
  return a.records +
         ((std::size_t(it.record) + (row - it.row)) * a.heads + head) * RecordFloats(D);
}

// The item's slots split over the waves, for up to 16 columns.
template<int D, class T, bool kRows32>
__device__ __forceinline__ void NarrowItem(const AttentionArgs& a, const lfm3_paged_item& it,
                                           int group, char* lds) {
  using Cols = Columns<D, T, kRows32, 1>;
  constexpr int kKeys = 4096 / D, KB = kKeys / 16;       // 8 KB of K and of V a wave
  constexpr int kLoads = kKeys * D * 2 / 1024;           // instructions a tile of K or V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = int(it.key_begin), end = int(it.key_end), g = int(it.kv_head);
  char* k_tile = lds + wave * 16384;
  char* v_tile = k_tile + 8192;
  const int step = kKeys * kWaves;
  int base = (begin & ~15) + wave * kKeys;
  RunPages<KB> pages = FetchPages<KB>(a.table, it.seq, base, end);
  const HeadRows k_rows = HeadRows::Of<D>(a.k_pages, a.table, a.kv_heads, g);
  const HeadRows v_rows = HeadRows::Of<D>(a.v_pages, a.table, a.kv_heads, g);
  unsigned offset[StageShape<D>::kPerRun];
#pragma unroll
  for (int i = 0; i < StageShape<D>::kPerRun; ++i)
    offset[i] = StageShape<D>::LaneOffset(i, lane);
  StageOwnTile<D, kKeys>(a.table, k_rows, pages, base, end, offset, k_tile);
  StageOwnTile<D, kKeys>(a.table, v_rows, pages, base, end, offset, v_tile);
  Cols cols;
  cols.Load(a, it, group, 0, lane);
  const Sight sight(it, a.window, int(it.slot), int(it.slot + it.rows) - 1);
  // One tile of the wave's; kOpen: every column sees all of it.
  const auto tile = [&]<bool kOpen>() {
    const RunPages<KB> next = FetchPages<KB>(a.table, it.seq, base + step, end);
    const unsigned holes = pages.Holes(a.table.pages);
    __builtin_amdgcn_s_waitcnt(WaitVm(kLoads));
    asm volatile("" ::: "memory");
    f4 s[1][KB];
    cols.template Scores<KB>(k_tile, lane, s);
    // The scores' reads are done before K's stage is filled again.
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    StageOwnTile<D, kKeys>(a.table, k_rows, next, base + step, end, offset, k_tile);
    typename Cols::V8 p[1][Cols::kParts][KB / 2];
    cols.template Softmax<KB, kOpen>(s, base, holes, lane, p);
    __builtin_amdgcn_s_waitcnt(WaitVm(kLoads));
    asm volatile("" ::: "memory");
    // A single row sees all that its tiles hold: the rest of them is zeros, but
    // for what a window leaves out of its first run.
    if (!kOpen && (it.rows > 1 || base < begin) && Cols::template Poisoned<KB>(v_tile, lane))
      cols.template OutputsApart<KB>(v_tile, lane, base, p);
    else
      cols.template Outputs<KB>(v_tile, lane, p);
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    StageOwnTile<D, kKeys>(a.table, v_rows, next, base + step, end, offset, v_tile);
    pages = next;
    base += step;
  };
  // The open tiles in a loop of their own: its state stays where it is.
  while (base < end) {
    while (base < end && base >= sight.whole_lo && base + kKeys - 1 <= sight.whole_hi &&
           !pages.Holes(a.table.pages))
      tile.template operator()<true>();
    if (base < end)
      tile.template operator()<false>();
  }
  // Loads past the span are still to land in the stages.
  __builtin_amdgcn_s_waitcnt(WaitVm(0));
  asm volatile("" ::: "memory");
  __syncthreads();
  // The waves' states meet in LDS: outputs [wave][column][D + 4], then maxima
  // and sums.
  constexpr int kPitch = D + 4;
  float* s_acc = reinterpret_cast<float*>(lds);
  float* s_m = s_acc + kWaves * 16 * kPitch;
  float* s_l = s_m + kWaves * 16;
  const int col = lane & 15, grp = lane >> 4;
  const float total = cols.Sum(0);
#pragma unroll
  for (int d = 0; d < Cols::kDims; ++d)
    *reinterpret_cast<f4*>(&s_acc[(wave * 16 + col) * kPitch + 16 * d + 4 * grp]) =
        cols.acc[0][d];
  if (grp == 0) {
    s_m[wave * 16 + col] = cols.m[0];
    s_l[wave * 16 + col] = total;
  }
  // Each column's scale, from the lanes that hold it.
  float* s_scale = s_l + kWaves * 16;
  if (wave == 0 && grp == 0)
    s_scale[col] = cols.scale[0];
  __syncthreads();
  const int c = tid / (D / 4), d = tid % (D / 4) * 4;
  if (c >= int(it.rows) * group)
    return;
  const std::size_t row = it.row + unsigned(c / group);
  const int head = g * group + c % group;
  const float scale = s_scale[c];
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    top = fmaxf(top, s_m[w * 16 + c]);
  const float shift = top == -INFINITY ? 0.0f : top;
  float l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = expf((s_m[w * 16 + c] - shift) * scale);
    l = fmaf(s_l[w * 16 + c], f, l);
    const f4 y = *reinterpret_cast<const f4*>(&s_acc[(w * 16 + c) * kPitch + d]);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = fmaf(y[i], f, x[i]);
  }
  if (it.parts > 1) {
    float* rec = Record<D>(a, it, row, head);
    *reinterpret_cast<f4*>(rec + d) = f4{x[0], x[1], x[2], x[3]};
    if (d == 0)
      *reinterpret_cast<f4*>(rec + D) = f4{top, l, scale, 0.0f};
    return;
  }
  StoreOutputs<D, T, kRows32, Cols::kPScale>(a, row, head, d, x, l, Gate(a, row, head));
  if (a.lse && d == 0)
    a.lse[row * a.heads + head] = top * scale + logf(l);
}

// The item's columns from `c_first` on split over the waves, 16 CT each.
template<int D, class T, bool kRows32, int CT>
__device__ __forceinline__ void WideItem(const AttentionArgs& a, const lfm3_paged_item& it,
                                         int group, int c_first, char* lds) {
  using Cols = Columns<D, T, kRows32, CT>;
  constexpr int KB = kWideKeys / 16, kTileBytes = kWideKeys * D * 2;
  constexpr int kLoads = kTileBytes / 1024 / kWaves;  // a wave's instructions a tile of K or V
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = int(it.key_begin), end = int(it.key_end), g = int(it.kv_head);
  // The wave's instructions: number wave + 8 u of the tile's, all at one place of
  // their runs.
  using Shape = StageShape<D>;
  static_assert(kWaves % Shape::kPerRun == 0, "one lane offset a wave");
  const HeadRows k_rows = HeadRows::Of<D>(a.k_pages, a.table, a.kv_heads, g);
  const HeadRows v_rows = HeadRows::Of<D>(a.v_pages, a.table, a.kv_heads, g);
  const unsigned offset = Shape::LaneOffset(wave, lane);
  const auto stage = [&](const RunPages<KB>& pages, int base, int st) {
    char* at = lds + st * 2 * kTileBytes + wave * 1024;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int run = (wave + kWaves * u) / Shape::kPerRun;
      const unsigned id = __builtin_amdgcn_readfirstlane(pages.Of(run));
      BufferToLds16(k_rows.Run<D>(a.table, id, base + 16 * run, end), offset, 0,
                    at + kWaves * u * 1024);
      BufferToLds16(v_rows.Run<D>(a.table, id, base + 16 * run, end), offset, 0,
                    at + kTileBytes + kWaves * u * 1024);
    }
  };
  const int first = begin & ~15;
  RunPages<KB> pages = FetchPages<KB>(a.table, it.seq, first, end);
  unsigned hole = pages.Holes(a.table.pages);  // of the tile at hand
  stage(pages, first, 0);
  pages = FetchPages<KB>(a.table, it.seq, first + kWideKeys, end);
  unsigned next_hole = pages.Holes(a.table.pages);
  stage(pages, first + kWideKeys, 1);
  pages = FetchPages<KB>(a.table, it.seq, first + 2 * kWideKeys, end);
  Cols cols;
  const int c0 = c_first + wave * 16 * CT;
  cols.Load(a, it, group, c0, lane);
  const int columns = int(it.rows) * group;
  const bool busy = c0 < columns;
  const Sight sight(it, a.window, int(it.slot) + c0 / group,
                    int(it.slot) + (min(c0 + 16 * CT, columns) - 1) / group);
  int st = 0, base = first;
  // One tile; kOpen: every column of the wave sees all of it.
  const auto tile = [&]<bool kOpen>() {
    // This tile's loads have landed (the next tile's may be in flight); after
    // the barrier every wave's have, and the stage of the tile before is free.
    __builtin_amdgcn_s_waitcnt(WaitVm(2 * kLoads));
    BlockBarrier();
    stage(pages, base + 2 * kWideKeys, st == 0 ? 2 : st - 1);
    const unsigned later_hole = pages.Holes(a.table.pages);
    pages = FetchPages<KB>(a.table, it.seq, base + 3 * kWideKeys, end);
    if (kOpen || (busy && base <= sight.reach_hi && base + kWideKeys > sight.reach_lo)) {
      const char* k_tile = lds + st * 2 * kTileBytes;
      const char* v_tile = k_tile + kTileBytes;
      f4 s[CT][KB];
      cols.template Scores<KB>(k_tile, lane, s);
      typename Cols::V8 p[CT][Cols::kParts][KB / 2];
      cols.template Softmax<KB, kOpen>(s, base, hole, lane, p);
      if (!kOpen && Cols::template Poisoned<KB>(v_tile, lane))
        cols.template OutputsApart<KB>(v_tile, lane, base, p);
      else
        cols.template Outputs<KB>(v_tile, lane, p);
    }
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    st = st == 2 ? 0 : st + 1;
    hole = next_hole;
    next_hole = later_hole;
    base += kWideKeys;
  };
  // The open tiles in a loop of their own: its state stays where it is. (Every
  // wave passes one barrier a tile, whichever loop it is in.)
  while (base < end) {
    while (busy && base < end && base >= sight.whole_lo &&
           base + kWideKeys - 1 <= sight.whole_hi && !hole)
      tile.template operator()<true>();
    if (base < end)
      tile.template operator()<false>();
  }
  // Loads past the span must not land after the block has ended.
  __builtin_amdgcn_s_waitcnt(WaitVm(0));
  asm volatile("" ::: "memory");
  const int grp = lane >> 4;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const float l = cols.Sum(ct);
    const unsigned c = unsigned(c0 + 16 * ct + (lane & 15)), r = c / unsigned(group);
    if (r >= it.rows)
      continue;
    const std::size_t row = it.row + r;
    const int head = g * group + int(c % unsigned(group));
    if (it.parts > 1) {
      float* rec = Record<D>(a, it, row, head);
#pragma unroll
      for (int d = 0; d < Cols::kDims; ++d)
        *reinterpret_cast<f4*>(rec + 16 * d + 4 * grp) = cols.acc[ct][d];
      if (grp == 0)
        *reinterpret_cast<f4*>(rec + D) = f4{cols.m[ct], l, cols.scale[ct], 0.0f};
      continue;
    }
    const float gate = Gate(a, row, head);
#pragma unroll
    for (int d = 0; d < Cols::kDims; ++d) {
      const float x[4] = {cols.acc[ct][d][0], cols.acc[ct][d][1], cols.acc[ct][d][2],
                          cols.acc[ct][d][3]};
      StoreOutputs<D, T, kRows32, Cols::kPScale>(a, row, head, 16 * d + 4 * grp, x, l,
                                                 gate);
    }
    if (a.lse && grp == 0)
      a.lse[row * a.heads + head] = cols.m[ct] * cols.scale[ct] + logf(l);
  }
}

// FP32 rows over BF16 pages of 128 dimensions: two column tiles a wave spill too
// much (96 registers of query parts, 64 of outputs, the scores and the
// probabilities' three parts), so a tile of more than 128 columns is two blocks
// of one each: 512 rows of 16 heads over 24,576 slots 256 us, 303 in one. (Over
// F16 pages, two parts, 215 and 201, though the one spills 79 registers; the kernels
// of 16-bit rows of 128 dimensions spill 22 and 23.)
template<int D, class T, bool kRows32>
constexpr bool kHalves = kRows32 && D == 128 && T::kType == LFM3_TYPE_BF16;

template<int D, class T, bool kRows32>
__launch_bounds__(kThreads, 2) __global__ void PagedAttentionKernel(AttentionArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const lfm3_paged_item it = UniformItem(a.items);
  const int group = a.heads / a.kv_heads;
  if (!Sound(a, it, group))
    return;
  const unsigned columns = it.rows * unsigned(group), c_first = blockIdx.y * kHalfColumns;
  if (c_first >= columns)
    return;
  if (columns <= kNarrowColumns)
    NarrowItem<D, T, kRows32>(a, it, group, lds);
  else if (kHalves<D, T, kRows32> || columns <= kHalfColumns)
    WideItem<D, T, kRows32, 1>(a, it, group, int(c_first), lds);
  else if constexpr (!kHalves<D, T, kRows32>)
    WideItem<D, T, kRows32, 2>(a, it, group, 0, lds);
}

// The records of a split tile's spans into its rows' outputs, the work shared
// out over the tile's items (and gridDim.y blocks of each, where there are few):
// item `part` takes that share of the columns. D / 4 lanes hold a record. Where a
// wave has columns enough, its groups of lanes take one each, twice (against
// groups that share a column's spans: 300 rows of 32 heads of 64 in two spans
// beside 7 decode rows, the call, 31 us and 38); else they share one's, and where
// there are fewer columns than waves two or four waves do. The loads of several
// spans and columns are in flight at once: what bounds a merge is its
// round trips to memory (the records come from other XCDs), and the dispatch of
// its waves (8 decode rows: 4.3 us in 448 blocks, 5.9 in 2016, 10.7 in 8064; 77
// rows over 3000 slots, the call: 20.0 us with kMergeBlocks 512, 18.8 with 768,
// 19.6 with 1024).
// Lanes' and waves' sums add in a fixed order.
constexpr int kMergeWaves = 4, kMergeThreads = 64 * kMergeWaves;
constexpr std::uint32_t kMergeBlocks = 768;

// A softmax state: an unnormalized output's four values, its maximum and sum.
struct MergeState {
  float top = -INFINITY, l = 0.0f;
  f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
  // Joined with another, this one's terms first; scale: of maxima, in base 2.
  __device__ __forceinline__ void Join(float top2, float l2, f4 x2, float scale) {
    const float next = fmaxf(top, top2), shift = next == -INFINITY ? 0.0f : next;
    const float w = __builtin_amdgcn_exp2f((top - shift) * scale);
    const float w2 = __builtin_amdgcn_exp2f((top2 - shift) * scale);
    top = next;
    l = l * w + l2 * w2;
    x = x * w + x2 * w2;
  }
};

template<int D, class T, bool kRows32>
__launch_bounds__(kMergeThreads) __global__ void PagedMergeKernel(AttentionArgs a) {
  constexpr int kLanes = D / 4, kSpans = 64 / kLanes;  // spans a wave takes at a time
  constexpr float kLog2e = 1.44269504088896341f;
  __shared__ f4 s_out[kMergeWaves][kLanes];
  __shared__ float2 s_state[kMergeWaves];
  const lfm3_paged_item it = UniformItem(a.items);
  const int group = a.heads / a.kv_heads, parts = int(it.parts);
  if (parts < 2 || !Sound(a, it, group))
    return;
  // The tile's first record; Sound() has bounded this item's own.
  const std::uint32_t before = it.part * it.rows;
  if (it.parts > kMaxParts || it.record < before ||
      std::uint64_t(it.record - before) + std::uint64_t(it.parts) * it.rows > a.max_records)
    return;
  const int columns = int(it.rows) * group;
  const int slice = int(it.part * gridDim.y + blockIdx.y), slices = parts * int(gridDim.y);
  const int begin = columns * slice / slices, end = columns * (slice + 1) / slices;
  if (begin == end)
    return;
  const int lane = threadIdx.x & 63, d = lane % kLanes * 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const std::size_t step = std::size_t(it.rows) * a.heads * RecordFloats(D);
  const auto record = [&](int c) {
    const std::size_t r = unsigned(c) / unsigned(group);
    return a.records + ((std::size_t(it.record - before) + r) * a.heads +
                        unsigned(int(it.kv_head) * group + c % group)) * RecordFloats(D);
  };
  const auto gate = [&](int c) {
    return Gate(a, it.row + unsigned(c / group), int(it.kv_head) * group + c % group);
  };
  const auto finish = [&](int c, bool mine, const MergeState& m, float scale, float raw) {
    const std::size_t row = it.row + unsigned(c / group);
    const int head = int(it.kv_head) * group + c % group;
    const float out[4] = {m.x[0], m.x[1], m.x[2], m.x[3]};
    if (mine)
      StoreOutputs<D, T, kRows32, Columns<D, T, kRows32, 1>::kPScale>(a, row, head, d, out, m.l,
                                                                      raw);
    if (a.lse && mine && d == 0)
      a.lse[row * a.heads + head] = m.top * scale + logf(m.l);
  };
  // Column c (clamped to the last one) over the spans first, first + stride, ...,
  // four in flight, and over the lanes that hold the same dimensions.
  const auto walk = [&](int c, int first, int stride, MergeState& m, float& scale, float& raw) {
    constexpr int B = 4;
    const float* rec = record(min(c, end - 1));
    scale = rec[D + 2];
    raw = gate(min(c, end - 1));
    for (int p0 = first + lane / kLanes; p0 < parts; p0 += B * stride) {
      f4 y[B];
      float2 ml[B];
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const float* s = rec + std::size_t(min(p0 + j * stride, parts - 1)) * step;
        y[j] = *reinterpret_cast<const f4*>(s + d);
        ml[j] = *reinterpret_cast<const float2*>(s + D);
      }
#pragma unroll
      for (int j = 0; j < B; ++j)
        if (p0 + j * stride < parts)
          m.Join(ml[j].x, ml[j].y, y[j], scale * kLog2e);
    }
#pragma unroll
    for (int k = kLanes; k < 64; k <<= 1) {
      // On both sides the lower lane's terms first.
      MergeState low, high;
      const float top2 = __shfl_xor(m.top, k), l2 = __shfl_xor(m.l, k);
      f4 x2;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x2[i] = __shfl_xor(m.x[i], k);
      const bool upper = lane & k;
      low.top = upper ? top2 : m.top;
      low.l = upper ? l2 : m.l;
      high.top = upper ? m.top : top2;
      high.l = upper ? m.l : l2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        low.x[i] = upper ? x2[i] : m.x[i];
        high.x[i] = upper ? m.x[i] : x2[i];
      }
      low.Join(high.top, high.l, high.x, scale * kLog2e);
      m = low;
    }
  };
  const int share = end - begin;
  if (share >= 2 * kMergeWaves) {
    // A column to a group of lanes, two after another, four spans of each in
    // flight; nothing crosses lanes.
    constexpr int U = 2, B = 4, kWave = kSpans * U;
    for (int c0 = begin + wave * kWave; c0 < end; c0 += kMergeWaves * kWave) {
      MergeState m[U];
      const float* rec[U];
      float scale[U], raw[U];
      int c[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        c[u] = c0 + u * kSpans + lane / kLanes;
        rec[u] = record(min(c[u], end - 1));
        scale[u] = rec[u][D + 2];
        raw[u] = gate(min(c[u], end - 1));
      }
      for (int p0 = 0; p0 < parts; p0 += B) {
        f4 y[U][B];
        float2 ml[U][B];
#pragma unroll
        for (int j = 0; j < B; ++j)
          if (p0 + j < parts)
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const float* s = rec[u] + std::size_t(p0 + j) * step;
              y[u][j] = *reinterpret_cast<const f4*>(s + d);
              ml[u][j] = *reinterpret_cast<const float2*>(s + D);
            }
#pragma unroll
        for (int j = 0; j < B; ++j)
          if (p0 + j < parts)
#pragma unroll
            for (int u = 0; u < U; ++u)
              m[u].Join(ml[u][j].x, ml[u][j].y, y[u][j], scale[u] * kLog2e);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c[u] < end)
          finish(c[u], true, m[u], scale[u], raw[u]);
    }
    return;
  }
  const int team = share >= 4 ? 1 : share >= 2 ? 2 : 4;  // waves a column
  for (int c0 = begin; c0 < end; c0 += kMergeWaves / team) {
    const int c = c0 + wave / team;
    MergeState m;
    float scale, raw;
    walk(c, wave % team * kSpans, team * kSpans, m, scale, raw);
    if (team > 1) {  // uniform over the block
      if (lane < kLanes)
        s_out[wave][lane] = m.x;
      if (lane == 0)
        s_state[wave] = make_float2(m.top, m.l);
      __syncthreads();
      m = MergeState();
      for (int w = wave / team * team; w < (wave / team + 1) * team; ++w)
        m.Join(s_state[w].x, s_state[w].y, s_out[w][lane % kLanes], scale * kLog2e);
      __syncthreads();  // read before the next columns' states are written
    }
    if (c < end && wave % team == 0)
      finish(c, lane < kLanes, m, scale, raw);
  }
}

// Items of a launch: a grid has less than 2^32 threads in x.
constexpr std::uint32_t kMaxBlocks = 1u << 22;

template<int D, class T, bool kRows32>
int LaunchKernels(AttentionArgs a, std::uint32_t n_items, hipStream_t s) {
  constexpr std::size_t kLds = std::size_t(kWaves) * 16384;
  static_assert(kLds >= kStages * 2 * kWideKeys * D * 2, "the wide ring fits");
  static_assert(kLds >= (kWaves * 16 * (D + 4) + 2 * kWaves * 16 + 16) * sizeof(float),
                "the narrow merge fits");
  const auto kernel = PagedAttentionKernel<D, T, kRows32>;
  const int e = HipStatus(
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                          hipFuncAttributeMaxDynamicSharedMemorySize, int(kLds)),
      "LFM3 paged attention shared memory");
  if (e)
    return e;
  const lfm3_paged_item* const items = a.items;
  for (std::uint32_t at = 0; at < n_items; at += kMaxBlocks) {
    a.items = items + at;
    kernel<<<dim3(std::min(n_items - at, kMaxBlocks), kHalves<D, T, kRows32> ? 2 : 1), kThreads,
             kLds, s>>>(a);
  }
  // After every item's records.
  for (std::uint32_t at = 0; a.max_records && at < n_items; at += kMaxBlocks) {
    a.items = items + at;
    PagedMergeKernel<D, T, kRows32><<<dim3(std::min(n_items - at, kMaxBlocks),
                                           std::clamp(kMergeBlocks / n_items, 1u, 32u)),
                                      kMergeThreads, 0, s>>>(a);
  }
  return HipStatus(hipGetLastError(), "LFM3 paged attention launch");
}
template<int D, class T>
int Launch(const AttentionArgs& a, std::uint32_t n_items, bool rows32, hipStream_t s) {
  return rows32 ? LaunchKernels<D, T, true>(a, n_items, s)
                : LaunchKernels<D, T, false>(a, n_items, s);
}

// ---------------------------------------------------------------- the plan

constexpr std::uint32_t kSpanFloor = 256, kMaxItems = 4096, kCus = 256, kXcds = 8;
// What the plan reckons with, in microseconds: a slot of an item of up to 16
// columns (measured: 0.005 and 3 an item in tiles of a chunk, which share their
// slots in L2; 0.011 or 0.022 where every CU streams its own), of a tile of up to
// 128 columns and of a full one (0.021 to 0.024, and 0.028 to 0.036, by the
// dimension and the rows' type, which it does not know), an item beside its
// slots, a merge and each of its parts. Against a dearer narrow item (0.007 and
// 4) 128 rows of 32 heads over 4000 slots take 15.4 us, 22.4 so, beside 16 decode
// rows 30 and 40, 1500 rows over 4000 135 and 164; 24 decode rows of 8192 to
// 32,768 slots 196 and 189, their spans cut once less.
constexpr double kNarrowSlot = 0.005, kHalfSlot = 0.023, kWideSlot = 0.036, kItemCost = 3,
                 kMergeCost = 5, kPartCost = 0.1, kRecordCost = 0.0002;  // a (row, head)'s record

// Rows [row, row + rows) of a sequence and the slots they see.
struct Tile {
  std::uint32_t seq, row, rows, slot, first, end, parts, span, record;
  double cost;  // of a slot
};

// Rows of a tile of `columns` columns.
std::uint32_t TileRows(std::uint32_t group, std::uint32_t columns) {
  return std::max(1u, columns / group);
}

// A tile's spans of at most `span` slots (whole multiples of 64 from the
// tile's first 64-slot run on, of one length).
void Split(Tile& t, std::uint64_t span) {
  const std::uint64_t from = t.first / 64 * 64, keys = t.end - from;
  span = std::max<std::uint64_t>(span, (keys + kMaxParts - 1) / kMaxParts);
  const std::uint64_t parts = (keys + span - 1) / span;
  const std::uint64_t even = ((keys + parts - 1) / parts + 63) / 64 * 64;
  t.span = std::uint32_t(even);
  t.parts = std::uint32_t((keys + even - 1) / even);
}

// The estimated time of a plan that splits by `span`, and its items.
double Estimate(std::vector<Tile>& tiles, std::uint64_t span, std::uint32_t group,
                std::uint32_t kv_heads, std::uint64_t& items) {
  double total = 0, longest = 0, records = 0;
  std::uint32_t parts = 1;
  items = 0;
  for (Tile& t : tiles) {
    Split(t, span);
    items += std::uint64_t(t.parts) * kv_heads;
    total += (double(t.end - t.first) * t.cost + kItemCost * t.parts) * kv_heads;
    longest = std::max(longest, std::min<double>(t.span, t.end - t.first) * t.cost + kItemCost);
    parts = std::max(parts, t.parts);
    records += t.parts > 1 ? double(t.parts) * t.rows * group * kv_heads : 0;
  }
  const double merge =
      parts > 1 ? kMergeCost + kPartCost * parts + kRecordCost * records : 0;
  return merge + (items <= kCus ? longest : std::max(longest, total / kCus + longest / 2));
}

int Plan(const std::uint32_t* starts, const std::uint32_t* lengths, std::uint32_t seqs,
         std::uint32_t group, std::uint32_t kv_heads, std::uint32_t window,
         lfm3_paged_item* items, std::uint32_t max_items) {
  // Tiles of 256 columns read their slots once for all of them; of 128, where
  // those do not fill the device, they make twice the blocks; of 16, whose
  // slots are split over a block's waves, they answer short spans soonest: 77
  // rows of 4 heads each that see 256 slots 9.2 us, 21.5 in tiles of 128; over
  // 1000 to 1077 slots 12.2 and 20.1; 512 rows without history 18.3 and 25.0.
  std::vector<Tile> tiles, trial;
  std::uint64_t best_span = 0, count = 0;
  double best = 0;
  for (const std::uint32_t columns : {kTileColumns, kHalfColumns, kNarrowColumns}) {
    const std::uint32_t most = TileRows(group, columns);
    std::uint64_t longest = 0;
    trial.clear();
    for (std::uint32_t s = 0; s < seqs; ++s) {
      const std::uint32_t rows = starts[s + 1] - starts[s];
      for (std::uint32_t r = 0; r < rows; r += most) {
        Tile t{};
        t.seq = s;
        t.row = starts[s] + r;
        t.rows = std::min(most, rows - r);
        t.slot = lengths[s] - rows + r;
        t.first = window && t.slot + 1 > window ? t.slot + 1 - window : 0;
        t.end = t.slot + t.rows;
        const std::uint32_t c = t.rows * group;
        t.cost = c <= kNarrowColumns ? kNarrowSlot : c <= kHalfColumns ? kHalfSlot : kWideSlot;
        longest = std::max<std::uint64_t>(longest, t.end - t.first);
        trial.push_back(t);
      }
    }
    if (trial.empty())
      return 0;
    if (columns == kNarrowColumns && std::uint64_t(trial.size()) * kv_heads > kMaxItems)
      break;  // no span would fit
    const std::uint64_t whole = std::max<std::uint64_t>(longest + 64, kSpanFloor);
    std::uint64_t span = kSpanFloor, chosen = 0;
    for (bool last = false; !last; span = (span * 9 / 8 + 63) / 64 * 64) {
      last = span >= whole;
      const double e = Estimate(trial, span, group, kv_heads, count);
      const bool fits = columns == kNarrowColumns
                            ? count <= kMaxItems
                            : last || count <= kMaxItems + std::uint64_t(trial.size()) * kv_heads;
      if (fits && (best == 0 || e < best)) {
        best = e;
        chosen = span;
      }
    }
    if (chosen) {
      best_span = chosen;
      tiles.swap(trial);
    }
  }
  Estimate(tiles, best_span, group, kv_heads, count);
  if (count > max_items)
    return Fail(LFM3_E_INVALID, "LFM3 paged attention plan exceeds its item list");
  std::uint64_t record = 0;
  for (Tile& t : tiles)
    if (t.parts > 1) {
      t.record = std::uint32_t(record);
      record += std::uint64_t(t.parts) * t.rows;
    }
  if (record > 0xffffffffu)
    return Fail(LFM3_E_INVALID, "LFM3 paged attention plan has too many records");
  // A run: the tiles of one sequence that walk the same span of one KV head.
  struct Run {
    std::uint32_t first, tiles, part, kv_head;
    double cost;
  };
  std::vector<Run> runs;
  for (std::uint32_t i = 0; i < tiles.size();) {
    std::uint32_t end = i;
    std::uint32_t parts = 0;
    for (; end < tiles.size() && tiles[end].seq == tiles[i].seq; ++end)
      parts = std::max(parts, tiles[end].parts);
    for (std::uint32_t p = 0; p < parts; ++p)
      for (std::uint32_t g = 0; g < kv_heads; ++g)
        runs.push_back(Run{i, end - i, p, g, tiles[i].span * tiles[i].cost * (end - i)});
    i = end;
  }
  // Blocks go to the XCDs in turn: each run to the XCD with the least so far,
  // the longest first; an XCD whose list ends takes from the longest list.
  std::stable_sort(runs.begin(), runs.end(),
                   [](const Run& a, const Run& b) { return a.cost > b.cost; });
  std::vector<lfm3_paged_item> queue[kXcds];
  double load[kXcds] = {};
  for (const Run& run : runs) {
    const auto x = std::size_t(std::min_element(load, load + kXcds) - load);
    load[x] += run.cost;
    for (std::uint32_t j = 0; j < run.tiles; ++j) {
      const Tile& t = tiles[run.first + j];
      if (run.part >= t.parts)
        continue;
      const std::uint64_t from = t.first / 64 * 64;
      lfm3_paged_item it{};
      it.seq = t.seq;
      it.row = t.row;
      it.rows = t.rows;
      it.slot = t.slot;
      it.key_begin = std::max(t.first, std::uint32_t(from + std::uint64_t(run.part) * t.span));
      it.key_end = std::uint32_t(
          std::min<std::uint64_t>(from + (std::uint64_t(run.part) + 1) * t.span, t.end));
      it.part = run.part;
      it.parts = t.parts;
      it.record = t.parts > 1 ? t.record + run.part * t.rows : 0;
      it.kv_head = run.kv_head;
      queue[x].push_back(it);
    }
  }
  std::size_t at[kXcds] = {};
  for (std::uint32_t n = 0; n < count; ++n) {
    std::size_t x = n % kXcds;
    if (at[x] == queue[x].size())
      for (std::size_t y = 0; y < kXcds; ++y)
        if (queue[y].size() - at[y] > queue[x].size() - at[x])
          x = y;
    items[n] = queue[x][at[x]++];
  }
  return int(count);
}

}  // namespace
}  // namespace lfm3amd

using namespace lfm3amd;

extern "C" {

int lfm3_paged_attention_plan(const std::uint32_t* starts, const std::uint32_t* lengths,
                              std::uint32_t seqs, std::uint32_t heads, std::uint32_t kv_heads,
                              std::uint32_t window, lfm3_paged_item* items,
                              std::uint32_t max_items) {
  if (!starts || !lengths || !items || !kv_heads || !heads || heads % kv_heads ||
      heads / kv_heads > kPagedMaxGroup || kv_heads > 65535 / kPagedMaxGroup)
    return Fail(LFM3_E_INVALID, "invalid LFM3 paged attention plan");
  for (std::uint32_t s = 0; s < seqs; ++s)
    if (starts[s + 1] < starts[s] || starts[s + 1] > 0x7fffffffu / kPagedMaxGroup ||
        lengths[s] > kMaxLength || lengths[s] < starts[s + 1] - starts[s])
      return Fail(LFM3_E_INVALID, "invalid LFM3 paged attention plan: starts or lengths");
  try {
    return Plan(starts, lengths, seqs, heads / kv_heads, kv_heads, window, items, max_items);
  } catch (const std::bad_alloc&) {
    return Fail(LFM3_E_NOMEM, "out of host memory");
  }
}

std::size_t lfm3_paged_attention_max_items(std::uint32_t rows, std::uint32_t seqs,
                                           std::uint32_t max_length, std::uint32_t heads,
                                           std::uint32_t kv_heads) {
  if (!kv_heads || !heads || heads % kv_heads || heads / kv_heads > kPagedMaxGroup)
    return 0;
  const auto tiles = [&](std::uint32_t columns) {
    return (rows / TileRows(heads / kv_heads, columns) + std::size_t(std::min(rows, seqs))) *
           kv_heads;
  };
  const std::size_t spans = std::clamp<std::size_t>(
      (std::size_t(max_length) + 64 + kSpanFloor - 1) / kSpanFloor, 1, kMaxParts);
  const std::size_t half = tiles(kHalfColumns), narrow = tiles(kNarrowColumns);
  return std::max(std::min<std::size_t>(kMaxItems + half, half * spans),
                  std::min<std::size_t>(kMaxItems, narrow * spans));
}

std::size_t lfm3_paged_attention_workspace_bytes(const lfm3_paged_item* items,
                                                 std::uint32_t n_items, std::uint32_t heads,
                                                 std::uint32_t dim) {
  std::size_t records = 0;
  for (std::uint32_t i = 0; items && i < n_items; ++i)
    if (items[i].parts > 1)
      records = std::max(records, std::size_t(items[i].record) + items[i].rows);
  return records * RecordBytes(heads, dim);
}

int lfm3_paged_attention(const lfm3_paged_cache* cache, const lfm3_paged_batch* batch,
                         const lfm3_paged_item* items, std::uint32_t n_items, const void* q,
                         std::uint32_t ldq, const float* gate, std::uint32_t ldg, void* out,
                         std::uint32_t ldo, std::uint32_t row_type, float* lse,
                         std::uint32_t heads, std::uint32_t window, void* workspace,
                         std::size_t workspace_bytes, void* stream) {
  int e = CheckPagedCache(cache);
  if (!e)
    e = CheckPagedBatch(batch);
  if (!e)
    e = CheckPagedRows(*cache, heads, row_type, q, ldq);
  if (!e)
    e = CheckPagedRows(*cache, heads, row_type, out, ldo);
  if (e)
    return e;
  if (!items || (gate && ldg < heads) || (workspace_bytes && !workspace) ||
      !Aligned16(workspace))
    return Fail(LFM3_E_INVALID, "invalid LFM3 paged attention");
  if (!n_items)
    return LFM3_OK;
  AttentionArgs a{q, ldq, gate, ldg, out, ldo, lse, static_cast<const Half*>(cache->k),
                  static_cast<const Half*>(cache->v),
                  PageTable{batch->tables, batch->table_stride, cache->pages,
                            PageShift(cache->page)},
                  items, static_cast<float*>(workspace), 0, batch->seqs, batch->rows, window,
                  int(heads), int(cache->kv_heads)};
  a.max_records = std::uint32_t(
      std::min<std::size_t>(workspace_bytes / RecordBytes(heads, cache->dim), 0xffffffffu));
  const auto s = static_cast<hipStream_t>(stream);
  const bool rows32 = row_type == LFM3_TYPE_F32, half = cache->type == LFM3_TYPE_F16;
  if (cache->dim == 128)
    return half ? Launch<128, F16Pages>(a, n_items, rows32, s)
                : Launch<128, Bf16Pages>(a, n_items, rows32, s);
  return half ? Launch<64, F16Pages>(a, n_items, rows32, s)
              : Launch<64, Bf16Pages>(a, n_items, rows32, s);
}

}  // extern "C"
