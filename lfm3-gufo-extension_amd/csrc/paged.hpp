// What the paged cache's operators share: the element types of pages, the
// cache and batch as kernels take them, and the checks of their arguments.
#ifndef LFM3_AMD_PAGED_HPP_
#define LFM3_AMD_PAGED_HPP_
#include "common.hpp"

namespace lfm3amd {

constexpr std::uint32_t kPagedMaxGroup = 64;
constexpr std::uint32_t kMaxLength = 1u << 30;  // slots of a sequence

// The 16-bit formats of pages and rows: conversions (to nearest even) and the
// matrix instruction of 16 x 16 outputs over 32 products each.
struct F16Pages {
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  static constexpr std::uint32_t kType = LFM3_TYPE_F16;
  static __device__ __forceinline__ float Load(unsigned bits) { return HalfBitsToFloat(bits); }
  static __device__ __forceinline__ Half Round(float x) { return FloatToHalfBits(x); }
  static __device__ __forceinline__ f4 Mfma(V8 a, V8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
struct Bf16Pages {
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  static constexpr std::uint32_t kType = LFM3_TYPE_BF16;
  static __device__ __forceinline__ float Load(unsigned bits) {
    return __uint_as_float(bits << 16);
  }
  static __device__ __forceinline__ Half Round(float x) {
    return __builtin_bit_cast(Half, static_cast<__bf16>(x));
  }
  static __device__ __forceinline__ f4 Mfma(V8 a, V8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// Element i of rows that are FP32 (kRows32) or the pages' type.
template<class T, bool kRows32>
__device__ __forceinline__ void StoreRow(void* p, std::size_t i, float x) {
  if constexpr (kRows32)
    static_cast<float*>(p)[i] = x;
  else
    static_cast<Half*>(p)[i] = T::Round(x);
}

template<class V8>
__device__ __forceinline__ V8 Pack4(const unsigned (&w)[4]) {
  return __builtin_bit_cast(V8, w);
}

// A query row of one head as the B operand of S^T = K Q^T: lane L holds
// dimensions 32 s + 8 (L / 16) .. + 7 of column L % 16 (its own row). FP32 rows
// keep their accuracy: the row, scaled by the power of two that brings its
// largest value to [2^14, 2^15), splits into two F16 parts that add up to it
// within 2^-21 of that value; for BF16 pages, unscaled, into three BF16 parts
// (within 2^-24 of each value). Products of parts are exact in FP32. Rows of
// the pages' type are one part.
template<int D, class T, bool kRows32>
struct Query {
  static constexpr bool kHalf = T::kType == LFM3_TYPE_F16;
  static constexpr int kParts = kRows32 ? (kHalf ? 2 : 3) : 1, kSteps = D / 32;
  uint4 raw[kSteps][kRows32 ? 2 : 1];

  // `at`: the head's first element. (A column without a row reads another's:
  // what it makes of it goes nowhere. A select here would wait for the loads.)
  __device__ __forceinline__ void Load(const void* rows, std::size_t at, int lane) {
    constexpr std::size_t kSize = kRows32 ? 4 : 2;
    const char* src = static_cast<const char*>(rows) + (at + 8 * (lane >> 4)) * kSize;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < (kRows32 ? 2 : 1); ++i)
        raw[s][i] = *reinterpret_cast<const uint4*>(src + 32 * kSize * s + 16 * i);
  }
  // The parts, and the scale of their scores (1 / sqrt(D) and the power of two).
  __device__ __forceinline__ void Split(typename T::V8 (&q)[kParts][kSteps], float& scale) const {
    constexpr float kRoot = D == 128 ? 0.08838834764831845f : 0.125f;
    if constexpr (!kRows32) {
      scale = kRoot;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        q[0][s] = __builtin_bit_cast(typename T::V8, raw[s][0]);
    } else {
      float x[kSteps][8], top = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const unsigned w[8] = {raw[s][0].x, raw[s][0].y, raw[s][0].z, raw[s][0].w,
                               raw[s][1].x, raw[s][1].y, raw[s][1].z, raw[s][1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[s][i] = __uint_as_float(w[i]);
          top = fmaxf(top, fabsf(x[s][i]));
        }
      }
      // Kept where both 2^e and 2^-e / sqrt(D) are normal.
      const int e = kHalf ? min(max(RowExponent(MaxXor32(MaxXor16(top))), -113), 100) : 0;
      scale = ldexpf(kRoot, -e);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        unsigned w[kParts][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float r0 = ldexpf(x[s][2 * i], e), r1 = ldexpf(x[s][2 * i + 1], e);
#pragma unroll
          for (int p = 0; p < kParts; ++p) {
            const unsigned b0 = T::Round(r0), b1 = T::Round(r1);
            w[p][i] = b0 | (b1 << 16);
            r0 -= T::Load(b0);
            r1 -= T::Load(b1);
          }
        }
#pragma unroll
        for (int p = 0; p < kParts; ++p)
          q[p][s] = Pack4<typename T::V8>(w[p]);
      }
    }
  }
};

// A slot's place: its page and the offset there, or no page.
struct PageTable {
  const std::uint32_t* tables;
  std::uint32_t stride, pages;
  int shift;  // log2(slots a page)
  __device__ __forceinline__ std::uint32_t Page(std::uint32_t seq, std::uint32_t slot) const {
    const std::uint32_t at = slot >> shift;
    return at < stride ? tables[std::size_t(seq) * stride + at] : ~0u;
  }
};

// The pages of a tile's runs of 16 slots, in scalar registers.
template<int kRuns>
struct RunPages {
  unsigned id[kRuns];
  // Run `r` (uniform).
  __device__ __forceinline__ unsigned Of(int r) const {
    static_assert(kRuns == 4, "two bits");
    const unsigned a = r & 1 ? id[1] : id[0], b = r & 1 ? id[3] : id[2];
    return r & 2 ? b : a;
  }
  // Bit r: run r is on no page.
  __device__ __forceinline__ unsigned Holes(unsigned pages) const {
    unsigned h = 0;
#pragma unroll
    for (int r = 0; r < kRuns; ++r)
      h |= (id[r] < pages ? 0u : 1u) << r;
    return h;
  }
};
// Those from slot `base` on; none past the span's end. All operands are
// uniform: the constant address space makes these scalar loads, which the
// vector loads' wait counts do not see. An index past the table reads its last
// entry, which is then masked out (a select would become a branch around each
// load, and the loads would follow one another).
template<int kRuns>
__device__ __forceinline__ RunPages<kRuns> FetchPages(const PageTable& table, std::uint32_t seq,
                                                      int base, int end) {
  typedef const __attribute__((address_space(4))) std::uint32_t Constant;
  Constant* entries = (Constant*)(table.tables + std::size_t(seq) * table.stride);
  RunPages<kRuns> p;
  unsigned out[kRuns];
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    const unsigned t = unsigned(base + 16 * r), at = t >> table.shift;
    out[r] = 0u - unsigned(int(t) >= end || at >= table.stride);
    p.id[r] = entries[min(at, table.stride - 1)];
  }
#pragma unroll
  for (int r = 0; r < kRuns; ++r)
    p.id[r] |= out[r];
  return p;
}

// Segment `seg` of slot `key`'s row lies at segment seg ^ SlotSwizzle(key):
// 16 slots at one segment (K operands), or 16 slots at a pair (V operands),
// take all 64 banks once.
template<int D>
__device__ __forceinline__ int SlotSwizzle(int key) {
  return D == 128 ? key & 15 : (key >> 1) & 7;
}

// One KV head's rows in a pool: page p's begin p * stride bytes after `base`.
struct HeadRows {
  const char* base;
  unsigned stride;
  template<int D>
  static __device__ __forceinline__ HeadRows Of(const Half* pool, const PageTable& table,
                                                int kv_heads, int g) {
    const unsigned page_bytes = unsigned(D * 2) << table.shift;
    return HeadRows{reinterpret_cast<const char*>(pool) + std::size_t(unsigned(g)) * page_bytes,
                    unsigned(kv_heads) * page_bytes};
  }
  // The resource of the run of 16 slots from `slot` on, on page `id`: those
  // before `end`; none where the run is on no page, as one that begins at `end`
  // or later must be. All scalar.
  template<int D>
  __device__ __forceinline__ BufferResource Run(const PageTable& table, unsigned id, int slot,
                                                int end) const {
    const bool there = id < table.pages;
    const unsigned in = unsigned(slot) & ((1u << table.shift) - 1);
    const unsigned left = __builtin_amdgcn_readfirstlane(min(end - slot, 16));
    return MakeBuffer(base + std::size_t(there ? id : 0u) * stride + in * unsigned(D * 2),
                      there ? left * unsigned(D * 2) : 0u);
  }
};

// A staging instruction moves 64 16-byte segments, kRows slots of a run:
// instruction n of a tile slots kRows n .. of it. A lane's offset in the run is
// the same for every run.
template<int D>
struct StageShape {
  static constexpr int kSegments = D / 8, kRows = 64 / kSegments, kPerRun = 16 / kRows;
  static __device__ __forceinline__ unsigned LaneOffset(int n, int lane) {
    const int key = n % kPerRun * kRows + lane / kSegments;
    return unsigned(key * D * 2 + ((lane % kSegments) ^ SlotSwizzle<D>(key)) * 16);
  }
};

// A wave's whole tile of kKeys slots from `slot` on into its own stage; offset:
// LaneOffset of instructions 0 .. kPerRun - 1. Slots from `end` on, and runs on
// no page, read as zeros.
template<int D, int kKeys>
__device__ __forceinline__ void StageOwnTile(const PageTable& table, const HeadRows& rows,
                                             const RunPages<kKeys / 16>& pages, int slot, int end,
                                             const unsigned (&offset)[StageShape<D>::kPerRun],
                                             char* lds) {
#pragma unroll
  for (int r = 0; r < kKeys / 16; ++r) {
    const BufferResource res =
        rows.Run<D>(table, __builtin_amdgcn_readfirstlane(pages.id[r]), slot + 16 * r, end);
#pragma unroll
    for (int i = 0; i < StageShape<D>::kPerRun; ++i)
      BufferToLds16(res, offset[i], 0, lds + (r * StageShape<D>::kPerRun + i) * 1024);
  }
}

// S^T = K Q^T over KB runs of 16 slots of a staged tile and CT tiles of 16
// columns: lane L's value i of run kb is slot 16 kb + 4 (L / 16) + i of column L
// % 16. Every operand read of K feeds all columns and parts.
template<int D, class T, int CT, int KB, int kParts>
__device__ __forceinline__ void TileScores(const char* tile, int lane,
                                           const typename T::V8 (&q)[CT][kParts][D / 32],
                                           f4 (&s)[CT][KB]) {
  using V8 = typename T::V8;
  constexpr int kSteps = D / 32;
  const int col = lane & 15, grp = lane >> 4;
  // A run's operands are read while the run before it is multiplied: 512 FP32
  // rows of 16 heads over 24,576 F16 slots of 128 took 224 us so, 244 with the
  // order left to the compiler.
  V8 k[2][kSteps];
  const auto read = [&](int kb) {
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
      k[kb & 1][st] = *reinterpret_cast<const V8*>(
          tile + (16 * kb + col) * (D * 2) + ((4 * st + grp) ^ SlotSwizzle<D>(col)) * 16);
  };
  read(0);
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    if (kb + 1 < KB)
      read(kb + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      s[ct][kb] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int p = 0; p < kParts; ++p)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          s[ct][kb] = T::Mfma(k[kb & 1][st], q[ct][p][st], s[ct][kb]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

inline int PageShift(std::uint32_t page) {
  switch (page) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    case 256: return 8;
    default: return -1;
  }
}
inline bool Aligned16(const void* p) { return (reinterpret_cast<std::uintptr_t>(p) & 15u) == 0; }

// LFM3_OK, or a status with its message set.
inline int CheckPagedCache(const lfm3_paged_cache* c) {
  if (!c || !c->k || !c->v || (c->type != LFM3_TYPE_F16 && c->type != LFM3_TYPE_BF16) ||
      !c->pages || PageShift(c->page) < 0 || !c->kv_heads || (c->dim != 64 && c->dim != 128) ||
      c->kv_heads > 65535 / kPagedMaxGroup || c->pages > 0x7fffffffu)
    return Fail(LFM3_E_INVALID, "unsupported LFM3 paged cache");
  if (!Aligned16(c->k) || !Aligned16(c->v) || !Aligned16(c->weight))
    return Fail(LFM3_E_INVALID, "LFM3 paged cache is not aligned");
  return LFM3_OK;
}
inline int CheckPagedBatch(const lfm3_paged_batch* b) {
  if (!b || !b->tables || !b->table_stride || !b->starts || !b->lengths || !b->seqs ||
      b->seqs > 65535 || b->rows > 0x7fffffffu / kPagedMaxGroup)
    return Fail(LFM3_E_INVALID, "invalid LFM3 paged batch");
  return LFM3_OK;
}
// Rows of heads * dim elements, `ld` apart, with whole 16-byte steps.
inline int CheckPagedRows(const lfm3_paged_cache& c, std::uint32_t heads, std::uint32_t type,
                          const void* p, std::uint32_t ld) {
  if (!heads || heads % c.kv_heads || heads / c.kv_heads > kPagedMaxGroup)
    return Fail(LFM3_E_INVALID, "unsupported LFM3 paged attention heads");
  if (type != LFM3_TYPE_F32 && type != c.type)
    return Fail(LFM3_E_INVALID, "LFM3 paged rows are FP32 or the pages' type");
  if (!p || !Aligned16(p) || ld < heads * c.dim || ld % (type == LFM3_TYPE_F32 ? 4 : 8))
    return Fail(LFM3_E_INVALID, "LFM3 paged rows are missing, too short or not aligned");
  return LFM3_OK;
}

}  // namespace lfm3amd
#endif
