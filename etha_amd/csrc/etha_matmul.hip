// Matrix products on local shards, MI355X (gfx950): 8-bit integers with scales, and products grouped by expert.
//
// One tile kernel serves every product here: an output tile out[r, c] = sum_k P(r, k) * Q(c, k), where either operand may
// lie k-contiguous in memory or transposed (k as the memory row).  The matrix instructions take 16 bytes of k a lane for
// 16-bit and for 8-bit elements alike, so both types share every layout.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "etha_device.h"
#include "etha_internal.h"
#include "etha_reshard.h"

using etha_internal::fail;
using etha_internal::g_kernel_launches;
using namespace etha_device;

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Element types of the operands: the matrix instruction on 16 bytes of k a lane.
struct ElemBF16 {
  static constexpr int kEs = 2;
  typedef f32x4 acc;
  static __device__ acc mfma(u32x4 a, u32x4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
// fp16 values below 2^-14: the instruction takes them with all their bits, but lines the products of a sum up as if they had the
// exponent of 2^-14, so that a sum in which such a product is among the largest keeps fewer bits: off by up to 18 units of 2^-24
// of the sum of magnitudes where 2 are the most otherwise (two terms, 10^8 sums), which is at most 2^-38 of the other factor.
struct ElemF16 {
  static constexpr int kEs = 2;
  typedef f32x4 acc;
  static __device__ acc mfma(u32x4 a, u32x4 b, acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct ElemI8 {
  static constexpr int kEs = 1;
  typedef i32x4 acc;
  static __device__ acc mfma(u32x4 a, u32x4 b, acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
};

// A sum of products of integers, which is exact, with its scales and bias: written as a fused operation, so that every kernel
// gives the same bits.
__device__ inline float scaled(float sum, float scale, bool with_bias, float bias) {
  return with_bias ? __builtin_fmaf(sum, scale, bias) : sum * scale;
}

enum Kind : uint32_t {
  kPlain = 0,        // one product: P k-contiguous, Q k-contiguous
  kGroupRows = 1,    // rows of P belong to groups, a Q for each group, k-contiguous
  kGroupRowsT = 2,   // the same with Q transposed (k is the memory row)
  kGroupReduce = 3,  // the reduction runs over a group's rows: both operands transposed, an output for each group
};

struct MatmulArgs {
  const char* p;
  const char* q;
  void* out;
  int64_t p_stride, q_stride, q_group_stride;  // bytes
  int64_t out_stride, out_group_stride;        // elements
  uint32_t rows, cols, red;                    // kGroupReduce: red is the number of rows that offsets cut
  const int32_t* offsets;                      // n_groups + 1 entries
  uint32_t n_groups, zero_rest;
  const float* row_scale;                      // 8 bits
  const float* col_scale;
  const float* bias;
  uint32_t splits;                             // kGroupReduce: parts that a group's rows are cut into, each with an output
  int64_t split_stride;                        // of its own, in elements
};

// ---- groups --------------------------------------------------------------------------------------------------------
// offsets come from the device and are not trusted: each entry is taken as the largest of itself and those before it,
// within [0, rows], so that groups never overlap or leave the tensor.
struct GroupTile {
  uint32_t group, lo, hi, tile;  // group: n_groups for rows of no group (to be zeroed); lo..hi its rows
  bool found;
};

__device__ inline int clamped(const int32_t* offsets, uint32_t i, uint32_t rows) {
  const int v = offsets[i];
  return v < 0 ? 0 : (uint32_t)v > rows ? (int)rows : v;
}

// The `want`-th tile of TILE rows over all groups; with zero_rest the rows before the first and behind the last group
// form groups of their own.
template <int TILE>
__device__ inline GroupTile find_tile(const MatmulArgs& a, uint32_t want) {
  const uint32_t lane = threadIdx.x & 63, n = a.n_groups + 2;  // before, the groups, behind
  uint32_t carry_hi = 0, carry_tiles = 0;
  for (uint32_t base = 0; base < n; base += 64) {
    const uint32_t g = base + lane;
    uint32_t hi = g <= a.n_groups ? (uint32_t)clamped(a.offsets, g, a.rows) : a.rows;
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(hi, d);
      if (lane >= (uint32_t)d && o > hi) hi = o;
    }
    hi = hi > carry_hi ? hi : carry_hi;
    uint32_t lo = __shfl_up(hi, 1);
    if (lane == 0) lo = carry_hi;
    const bool rest = g == 0 || g == a.n_groups + 1;
    uint32_t tiles = g < n && (!rest || a.zero_rest) ? (hi - lo + TILE - 1) / TILE : 0;
    uint32_t inc = tiles;
    #pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(inc, d);
      if (lane >= (uint32_t)d) inc += o;
    }
    inc += carry_tiles;
    const uint64_t past = __ballot(inc > want);
    if (past) {
      const int l = __builtin_ctzll(past);
      GroupTile t;
      const uint32_t gg = base + l;
      t.group = gg == 0 || gg == a.n_groups + 1 ? a.n_groups : gg - 1;
      t.lo = __builtin_amdgcn_readlane(lo, l);
      t.hi = __builtin_amdgcn_readlane(hi, l);
      t.tile = want - (__builtin_amdgcn_readlane(inc, l) - __builtin_amdgcn_readlane(tiles, l));
      t.found = true;
      return t;
    }
    carry_hi = __builtin_amdgcn_readlane(hi, 63);
    carry_tiles = __builtin_amdgcn_readlane(inc, 63);
  }
  return GroupTile{0, 0, 0, 0, false};
}

// Rows [lo, hi) of one group.
__device__ inline void group_bounds(const MatmulArgs& a, uint32_t group, uint32_t* lo, uint32_t* hi) {
  const uint32_t lane = threadIdx.x & 63;
  int top = 0;
  for (uint32_t i = lane; i <= group; i += 64) {
    const int v = clamped(a.offsets, i, a.red);
    top = v > top ? v : top;
  }
  #pragma unroll
  for (int d = 32; d; d >>= 1) {
    const int o = __shfl_xor(top, d);
    top = o > top ? o : top;
  }
  top = __builtin_amdgcn_readfirstlane(top);
  const int end = clamped(a.offsets, group + 1, a.red);
  *lo = (uint32_t)top;
  *hi = (uint32_t)(end > top ? end : top);
}

// ---- staging -------------------------------------------------------------------------------------------------------
// A stage holds kStageBytes of k of both operands.  Where an operand lies k-contiguous in memory its LDS tile is ROWS rows
// of kStageBytes, read 16 bytes of k a lane; where it lies transposed (16-bit elements) the tile is the memory's own [k][ROWS],
// read with the transposing LDS load, which hands each of 16 lanes four k of one column.  Either tile is a sequence of
// 16-byte slots; which piece of memory a slot holds is permuted so that the lanes of one read touch all banks: by the row
// where 16 rows are read at one k, in 32-byte column groups by (k & 3, k >> 3) where 8 rows of k are read at one column.
constexpr int kStageBytes = 128;            // whole lines of memory: 64-byte pieces of rows were 10 % slower
constexpr uint32_t kOutside = 0x80000000u;  // an offset that no operand's tile reaches: reads there give zeros

template <typename E, bool TRANS_, int ROWS, int THREADS_>
struct Operand {
  static constexpr bool kTrans = TRANS_;
  static constexpr int kEs = E::kEs, kThreads = THREADS_;
  static constexpr int kStageK = kStageBytes / kEs;
  static constexpr int kBytes = ROWS * kStageBytes, kSlots = kBytes / 16, kPer = kSlots / kThreads;
  static constexpr int kPieces = kTrans ? ROWS / 8 : kStageBytes / 16;  // slots of an LDS row
  static_assert(kSlots % kThreads == 0 && kPer > 0, "every work-item stages the same number of slots");
  static_assert(kPer == 1 || kThreads / kPieces % 16 == 0, "all slots of a work-item hold the same piece of their rows");

  static __device__ uint32_t row_of(uint32_t slot) { return slot / kPieces; }
  static __device__ uint32_t swizzle(uint32_t row, uint32_t piece) {
    if constexpr (kTrans) return piece ^ ((((row & 3) | ((row >> 1) & 4)) << 1) & (kPieces - 1));
    else return piece ^ (row & 7);
  }
  static __device__ uint32_t piece_of(uint32_t slot) { return swizzle(row_of(slot), slot % kPieces); }

  // The 16 bytes of k that this lane needs of tile row r0 + (lane & 15), from k piece kp0 + (lane >> 4) of the stage.
  static __device__ u32x4 fragment(const char* lds, uint32_t r0, uint32_t kp0) {
    const uint32_t lane = threadIdx.x & 63;
    if constexpr (!kTrans) {
      const uint32_t r = r0 + (lane & 15);
      return *(const u32x4*)(lds + r * kStageBytes + swizzle(r, kp0 + (lane >> 4)) * 16);
    } else {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const uint32_t k = (kp0 + (lane >> 4)) * 8 + ((lane & 15) >> 2), col = r0 + (lane & 3) * 4;
      const char* p = lds + k * (ROWS * 2) + swizzle(k, col >> 3) * 16 + (col & 7) * 2;
      // rows k and k + 4 have the same permutation
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * ROWS * 2)));
      return u32x4{a.x, a.y, b.x, b.y};
    }
  }
};

__device__ inline uint32_t lds_address(const char* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }

// Straight from memory into LDS, 16 bytes a lane: for operands whose rows start at 16-byte addresses and, k-contiguous
// ones, hold whole 16-byte pieces of k.  The buffer descriptor ends with the operand tile's last word, so that whatever
// the tile reaches over reads as zero.  It has to be the whole word: memory is checked against the end word by word, and of
// one that lies across it nothing arrives, the last element of an odd width among it.  The other half of that word lies in
// the same 16 bytes of memory, and belongs to a column whose results are dropped.  The loads write no registers; the kernel
// waits for them by count.
template <typename OP>
struct DirectStage {
  static constexpr bool kDirect = true;
  uint32_t at[OP::kPer];
  uint32_t k_byte;   // where in the stage's k this lane's pieces lie (one place for all of them)
  const char* base;
  int64_t left;      // bytes from base to the end of the operand's tile
  uint32_t stride;
  uint32_t wave_at;  // where this wave's first slot lies in a stage

  __device__ void init(const char* tile, int64_t row_stride, uint32_t n_rows, uint32_t red) {
    base = tile;
    stride = (uint32_t)row_stride;
    left = OP::kTrans ? (int64_t)((int)red - 1) * row_stride + (int64_t)n_rows * 2
                      : (int64_t)((int)n_rows - 1) * row_stride + (int64_t)red * OP::kEs;
    left = (left + 3) & ~(int64_t)3;
    #pragma unroll
    for (int i = 0; i < OP::kPer; i++) {
      const uint32_t slot = threadIdx.x + i * OP::kThreads;
      at[i] = OP::row_of(slot) * stride + OP::piece_of(slot) * 16;
    }
    k_byte = OP::piece_of(threadIdx.x) * 16;
    wave_at = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
  }
  // The stage that begins at k0, into LDS, in kPer parts; past the end of k it brings zeros.
  u32x4 rsrc;
  uint32_t to, outside;
  __device__ void begin(char* lds, uint32_t k0, uint32_t red) {
    const uint64_t b = (uint64_t)base;
    const uint32_t size = left > 0x7fffffff ? 0x7fffffffu : left < 0 ? 0u : (uint32_t)left;
    rsrc = u32x4{(uint32_t)b, (uint32_t)(b >> 32) & 0xffffu, size, 0x00020000u};
    to = lds_address(lds) + wave_at;
    outside = 0;
    if constexpr (!OP::kTrans) outside = (int64_t)k_byte >= ((int64_t)red - (int64_t)k0) * OP::kEs ? kOutside : 0;
    const int64_t step = OP::kTrans ? (int64_t)OP::kStageK * stride : (int64_t)OP::kStageK * OP::kEs;
    base += step;
    left -= step;
  }
  // m0, where the load's place in LDS stands, is named as written: nothing else in these kernels uses it, and whatever a
  // compiler may make of them has to set it anew.  (The warning is about registers that are not kept across the statement.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
  __device__ void part(int i) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(to + i * OP::kThreads * 16), "v"(at[i] | outside), "s"(rsrc) : "memory", "m0");
  }
#pragma clang diagnostic pop
};

// n bytes (0 to 16) dropped at the low end, zeros in at the high end
__device__ inline u32x4 shift_bytes(u32x4 v, uint32_t n) {
  uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
  if (n >= 8) {
    lo = n >= 16 ? 0 : hi >> ((n - 8) * 8);
    hi = 0;
  } else if (n) {
    lo = lo >> (n * 8) | hi << (64 - n * 8);
    hi >>= n * 8;
  }
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// Through registers: any start, any distance, any length of rows from 16 bytes on.  The next stage's loads are in flight
// during a stage, so there are no branches about them: a piece that reaches over its row's end is loaded from 16 bytes
// before that end, and shifted into place when it is stored to LDS.
template <typename OP>
struct RegisterStage {
  static constexpr bool kDirect = false;
  u32x4 v[OP::kPer];
  const char* base;
  uint32_t stride, n_rows;
  uint32_t row0, across;  // this lane's first row (k where transposed) and where its pieces lie in a row, in bytes
  uint32_t shift, inside; // of the stage that is in the registers: bytes to drop, rows of k that there are
  bool odd;               // whether any of it has to be put in order

  static constexpr uint32_t kRowStep = OP::kThreads / OP::kPieces;

  __device__ void init(const char* tile, int64_t row_stride, uint32_t n_rows_, uint32_t) {
    base = tile;
    stride = (uint32_t)row_stride;
    n_rows = n_rows_;
    row0 = OP::row_of(threadIdx.x);
    across = OP::piece_of(threadIdx.x) * 16;
  }
  __device__ void load(uint32_t k0, uint32_t red) {
    if constexpr (!OP::kTrans) {
      const int left = (int)((red - k0) * OP::kEs) - (int)across;  // bytes of the row from this piece on
      shift = left >= 16 ? 0 : left > 0 ? 16 - left : 16;
      odd = k0 + OP::kStageK > red;
      const uint32_t at = left >= 16 ? k0 * OP::kEs + across : red * OP::kEs - 16;
      #pragma unroll
      for (int i = 0; i < OP::kPer; i++) {
        const uint32_t row = row0 + i * kRowStep;  // rows past the last repeat it; their results are dropped
        v[i] = load_raw<16>(base + ((row < n_rows ? row : n_rows - 1) * stride + at));
      }
    } else {
      const int left = (int)(n_rows * 2) - (int)across;
      shift = left >= 16 ? 0 : left > 0 ? 16 - left : 0;  // columns past the last: their results are dropped
      inside = red - k0 < OP::kStageK ? red - k0 : OP::kStageK;
      odd = inside < OP::kStageK || n_rows * 2 < OP::kPieces * 16;
      const char* from = base + (int64_t)k0 * stride + (left >= 16 ? (int)across : (int)(n_rows * 2) - 16);
      #pragma unroll
      for (int i = 0; i < OP::kPer; i++) {
        const uint32_t row = row0 + i * kRowStep;
        v[i] = load_raw<16>(from + (row < inside ? row : inside - 1) * stride);
      }
    }
  }
  __device__ void store(char* lds) {
    if (odd) {
      #pragma unroll
      for (int i = 0; i < OP::kPer; i++)
        v[i] = shift_bytes(v[i], OP::kTrans && row0 + i * kRowStep >= inside ? 16 : shift);
    }
    #pragma unroll
    for (int i = 0; i < OP::kPer; i++) *(u32x4*)(lds + (threadIdx.x + i * OP::kThreads) * 16) = v[i];
  }
};

// ---- the tile kernel -----------------------------------------------------------------------------------------------
// A tile of BM rows and BN columns, WM x WN waves, STAGES stages of kStageBytes of k in LDS.  The fragments of the next
// half of a stage are read while the matrix units work on this one's.  One barrier a stage, in front of its second half:
// every wave then has all it needs of the stage in registers, so that its LDS can take a stage further on.
template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
  static constexpr int kThreads = WM * WN * 64;
};

template <int N>
__device__ inline void wait_stage() {  // at most N loads into LDS outstanding; this wave's LDS reads done
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
}

struct Tile {
  const char *p, *q;
  int64_t out;  // offset of its group's results, in elements
  uint32_t row0, row_end, col0;
  uint32_t red;  // 0 also for rows of no group: they become zeros
  bool there;
};

// This workgroup's tile.
template <typename E, uint32_t KIND, typename S>
__device__ inline Tile locate(const MatmulArgs& a) {
  constexpr bool kTransP = KIND == kGroupReduce, kTransQ = KIND == kGroupReduce || KIND == kGroupRowsT;
  constexpr uint32_t kStageK = kStageBytes / E::kEs;
  Tile t = {};
  t.there = true;
  uint32_t id = blockIdx.x;
  const uint32_t col_tiles = (a.cols + S::BN - 1) / S::BN;
  // Workgroups go to the 8 XCDs in turn: each XCD takes a run of the tiles, so that its L2 sees operands again.  In a run
  // the tiles go down bands of kBand row tiles.  Groups of a sum over their rows cost as much as they have rows: there every
  // XCD takes a run of every group's tiles.
  constexpr uint32_t kBand = 4;
  const uint32_t n = KIND == kGroupReduce ? gridDim.x / a.n_groups : gridDim.x;
  const uint32_t group = KIND == kGroupReduce ? id / n : 0;
  id -= group * n;
  const uint32_t xcd = id & 7, each = n >> 3, more = n & 7;
  id = xcd * each + (xcd < more ? xcd : more) + (id >> 3);
  const uint32_t row_tiles = n / col_tiles, band = id / (kBand * col_tiles);
  const uint32_t in_band = row_tiles - band * kBand < kBand ? row_tiles - band * kBand : kBand;
  id -= band * kBand * col_tiles;
  const uint32_t row_id = band * kBand + id % in_band;
  t.col0 = id / in_band * S::BN;
  t.p = a.p;
  t.q = a.q;
  t.red = a.red;
  t.row0 = row_id * S::BM;
  t.row_end = a.rows;
  if constexpr (KIND == kGroupReduce) {
    uint32_t lo, hi;
    group_bounds(a, group, &lo, &hi);
    if (a.splits > 1) {  // this part's stages
      const uint32_t part = ((hi - lo + kStageK - 1) / kStageK + a.splits - 1) / a.splits * kStageK;
      const uint64_t from = (uint64_t)lo + (uint64_t)blockIdx.y * part;
      lo = from < hi ? (uint32_t)from : hi;
      hi = hi - lo > part ? lo + part : hi;
      t.out += (int64_t)blockIdx.y * a.split_stride;
    }
    t.red = hi - lo;
    t.p += (int64_t)lo * a.p_stride;
    t.q += (int64_t)lo * a.q_stride;
    t.out += (int64_t)group * a.out_group_stride;
  } else if constexpr (KIND != kPlain) {
    const GroupTile g = find_tile<S::BM>(a, row_id);
    t.there = g.found;
    t.row0 = g.lo + g.tile * S::BM;
    t.row_end = g.hi;
    if (g.group == a.n_groups) t.red = 0;
    else t.q += (int64_t)g.group * a.q_group_stride;
  }
  t.p += kTransP ? (int64_t)t.row0 * E::kEs : (int64_t)t.row0 * a.p_stride;
  t.q += kTransQ ? (int64_t)t.col0 * E::kEs : (int64_t)t.col0 * a.q_stride;
  return t;
}

template <typename E, uint32_t KIND, typename D, typename S, template <typename> class STAGE>
__global__ __launch_bounds__(S::kThreads) void etha_matmul_kernel(const MatmulArgs a) {
  typedef Operand<E, KIND == kGroupReduce, S::BM, S::kThreads> OpP;
  typedef Operand<E, KIND == kGroupReduce || KIND == kGroupRowsT, S::BN, S::kThreads> OpQ;
  constexpr bool kDirect = STAGE<OpP>::kDirect;
  constexpr int kStages = kDirect ? S::STAGES : 2, kFm = S::BM / S::WM / 16, kFn = S::BN / S::WN / 16;
  constexpr uint32_t kStageK = OpP::kStageK, kBytes = OpP::kBytes + OpQ::kBytes;
  __shared__ __align__(1024) char lds[kStages * kBytes];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t wr = wave / S::WN * (S::BM / S::WM), wc = wave % S::WN * (S::BN / S::WN);

  const Tile tile = locate<E, KIND, S>(a);
  if (!tile.there) return;
  STAGE<OpP> sp;
  STAGE<OpQ> sq;
  {
    const uint32_t n_rows = tile.row_end - tile.row0, n_cols = a.cols - tile.col0;
    sp.init(tile.p, a.p_stride, n_rows < S::BM ? n_rows : S::BM, tile.red);
    sq.init(tile.q, a.q_stride, n_cols < S::BN ? n_cols : S::BN, tile.red);
  }
  constexpr int kReads = kFm + kFn;
  u32x4 fp[kDirect ? 2 : 1][kFm], fq[kDirect ? 2 : 1][kFn];
  const auto read = [&](int set, const char* from, int half, int t) {
    if (t < kFn) fq[set][t] = OpQ::fragment(from + OpP::kBytes, wc + t * 16, half * 4);
    else fp[set][t - kFn] = OpP::fragment(from, wr + (t - kFn) * 16, half * 4);
  };
  typename E::acc acc[kFm][kFn] = {};
  if constexpr (kDirect) {
    constexpr int kParts = OpP::kPer + OpQ::kPer;
    // fragments to read in a row of matrix instructions: done well before the barrier waits for them
    constexpr int kReadRows = kFm * 3 / 4 > 0 ? kFm * 3 / 4 : 1, kReadsRow = (kReads + kReadRows - 1) / kReadRows;
    uint32_t next = 0;  // k of the first stage that is not on its way yet
    const auto begin = [&](char* to) {
      sp.begin(to, next, tile.red);
      sq.begin(to + OpP::kBytes, next, tile.red);
      next += kStageK;
    };
    const auto part = [&](int t) {
      if (t < OpP::kPer) sp.part(t);
      else sq.part(t - OpP::kPer);
    };
    if (tile.red) {
      #pragma unroll
      for (int s = 0; s < kStages; s++) {
        begin(lds + s * kBytes);
        #pragma unroll
        for (int t = 0; t < kParts; t++) part(t);
      }
      wait_stage<(kStages - 1) * kParts>();
      #pragma unroll
      for (int t = 0; t < kReads; t++) read(0, lds, 0, t);
      uint32_t use = 0;
      for (uint32_t k = 0; k < tile.red; k += kStageK) {
        const uint32_t then = use + kBytes == sizeof(lds) ? 0 : use + kBytes;
        #pragma unroll
        for (int h = 0; h < 2; h++) {
          if (h == 1) {
            wait_stage<(kStages - 2) * kParts>();
            begin(lds + use);  // past the end of k it brings zeros: the count of loads stays the same
          }
          // a row of matrix instructions, the next half's fragments and the loads of a stage further on, in turn: issued
          // in a row each of them would hold up the others
          #pragma unroll
          for (int i = 0; i < kFm; i++) {
            #pragma unroll
            for (int t = i * kReadsRow; t < (i + 1) * kReadsRow && t < kReads; t++) read(h ^ 1, lds + (h ? then : use), h ^ 1, t);
            #pragma unroll
            for (int j = 0; j < kFn; j++) acc[i][j] = E::mfma(fq[h][j], fp[h][i], acc[i][j]);
            if (h == 1) {
              #pragma unroll
              for (int t = i * kParts / kFm; t < (i + 1) * kParts / kFm; t++) part(t);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        use = then;
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into this LDS outlives the workgroup
    }
  } else if (tile.red) {
    sp.load(0, tile.red);
    sq.load(0, tile.red);
    sp.store(lds);
    sq.store(lds + OpP::kBytes);
    __syncthreads();
    uint32_t use = 0;
    for (uint32_t k = 0; k < tile.red; k += kStageK) {
      const uint32_t then = use ^ kBytes;
      const bool more = k + kStageK < tile.red;
      if (more) {
        sp.load(k + kStageK, tile.red);
        sq.load(k + kStageK, tile.red);
      }
      #pragma unroll
      for (int h = 0; h < 2; h++) {
        #pragma unroll
        for (int t = 0; t < kReads; t++) read(0, lds + use, h, t);
        #pragma unroll
        for (int i = 0; i < kFm; i++)
          #pragma unroll
          for (int j = 0; j < kFn; j++) acc[i][j] = E::mfma(fq[0][j], fp[0][i], acc[i][j]);
      }
      if (more) {
        sp.store(lds + then);
        sq.store(lds + then + OpP::kBytes);
      }
      __syncthreads();
      use = then;
    }
  }
  // a lane holds row (lane & 15) and four consecutive columns of each 16 x 16 block
  const uint32_t row_first = tile.row0 + wr + (lane & 15), col_first = tile.col0 + wc + (lane >> 4) * 4;
  typename D::bits* out = (typename D::bits*)a.out + tile.out;
  float col_scale[kFn][4], bias[kFn][4];
  if constexpr (E::kEs == 1) {
    #pragma unroll
    for (int j = 0; j < kFn; j++)
      #pragma unroll
      for (int c = 0; c < 4; c++) {
        const uint32_t col = col_first + j * 16 + c < a.cols ? col_first + j * 16 + c : a.cols - 1;
        col_scale[j][c] = a.col_scale[col];
        bias[j][c] = a.bias ? a.bias[col] : 0.f;
      }
  }
  // 16-bit results of two neighbouring blocks change places between the lanes, so that a lane stores 16 bytes and four of
  // them 64 bytes of a row, instead of 8 and 32
  constexpr bool kPairs = sizeof(typename D::bits) == 2 && kFn % 2 == 0;
  const auto store_tile = [&](auto whole) {
    #pragma unroll
    for (int i = 0; i < kFm; i++) {
      const uint32_t row = row_first + i * 16;
      float row_scale = 1.f;
      if constexpr (E::kEs == 1) row_scale = a.row_scale[whole || row < tile.row_end ? row : tile.row_end - 1];
      typename D::bits* to = out + (int64_t)row * a.out_stride;
      float v[kFn][4];
      #pragma unroll
      for (int j = 0; j < kFn; j++)
        #pragma unroll
        for (int c = 0; c < 4; c++) {
          if constexpr (E::kEs == 1) {
            v[j][c] = scaled((float)acc[i][j][c], row_scale * col_scale[j][c], a.bias != nullptr, bias[j][c]);
          } else {
            v[j][c] = acc[i][j][c];
          }
        }
      if constexpr (kPairs) {
        #pragma unroll
        for (int j = 0; j < kFn; j += 2) {
          u32x4 w;
          #pragma unroll
          for (int c = 0; c < 2; c++) {
            const uint32_t x = (uint32_t)D::from_f32(v[j][2 * c]) | (uint32_t)D::from_f32(v[j][2 * c + 1]) << 16;
            const uint32_t y = (uint32_t)D::from_f32(v[j + 1][2 * c]) | (uint32_t)D::from_f32(v[j + 1][2 * c + 1]) << 16;
            const u32x2 r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
            w[c] = r.x;
            w[2 + c] = r.y;
          }
          // groups of 16 lanes: columns 0..7 of block j, of block j + 1, then 8..15 of either
          const uint32_t col = tile.col0 + wc + j * 16 + (lane >> 4 & 1) * 16 + (lane >> 5) * 8;
          if (whole) {
            store_raw<16>(to + col, w);
          } else if (row < tile.row_end) {
            if (col + 8 <= a.cols) {
              store_raw<16>(to + col, w);
            } else {
              #pragma unroll
              for (int e = 0; e < 8; e++)
                if (col + e < a.cols) to[col + e] = (typename D::bits)(w[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
      } else if (whole || row < tile.row_end) {
        #pragma unroll
        for (int j = 0; j < kFn; j++)
          store_f32<D, 4>(to + col_first + j * 16, v[j], whole ? 4 : (int64_t)a.cols - (col_first + j * 16));
      }
    }
  };
  if (tile.row0 + S::BM <= tile.row_end && tile.col0 + S::BN <= a.cols) store_tile(std::true_type{});
  else store_tile(std::false_type{});
}

// ---- rows shorter than 16 bytes ------------------------------------------------------------------------------------
// A work-item an element: nothing here is worth a tile.
template <typename E>
__device__ inline typename std::conditional<E::kEs == 1, int, float>::type element(const char* p) {
  if constexpr (E::kEs == 1) return *(const int8_t*)p;
  else if constexpr (std::is_same_v<E, ElemBF16>) return BF16::to_f32(*(const uint16_t*)p);
  else return F16::to_f32(*(const uint16_t*)p);
}

template <typename E, uint32_t KIND, typename D>
__global__ __launch_bounds__(256) void etha_matmul_short_kernel(const MatmulArgs a) {
  constexpr bool kTransP = KIND == kGroupReduce, kTransQ = KIND == kGroupReduce || KIND == kGroupRowsT;
  const uint64_t groups = KIND == kGroupReduce ? a.n_groups : 1, count = groups * a.rows * a.cols;
  for (uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x; id < count; id += (uint64_t)gridDim.x * 256) {
    const uint32_t col = (uint32_t)(id % a.cols);
    const uint64_t row = id / a.cols % a.rows;
    const uint32_t g = (uint32_t)(id / a.cols / a.rows);
    const char *p = a.p, *q = a.q;
    uint32_t red = a.red;
    int64_t out = (int64_t)g * a.out_group_stride;
    if constexpr (KIND == kGroupReduce) {
      int lo = 0;
      for (uint32_t i = 0; i <= g; i++) {
        const int v = clamped(a.offsets, i, a.red);
        lo = v > lo ? v : lo;
      }
      const int hi = clamped(a.offsets, g + 1, a.red);
      red = hi > lo ? hi - lo : 0;
      p += (int64_t)lo * a.p_stride;
      q += (int64_t)lo * a.q_stride;
    } else if constexpr (KIND != kPlain) {
      uint32_t e = 0;  // the entries up to the row's own, which the largest so far never passes before
      while (e <= a.n_groups && (uint64_t)clamped(a.offsets, e, a.rows) <= row) e++;
      if (e == 0 || e > a.n_groups) {  // rows of no group
        if (!a.zero_rest) continue;
        red = 0;
      } else {
        q += (int64_t)(e - 1) * a.q_group_stride;
      }
    }
    p += kTransP ? (int64_t)row * E::kEs : (int64_t)row * a.p_stride;
    q += kTransQ ? (int64_t)col * E::kEs : (int64_t)col * a.q_stride;
    typename std::conditional<E::kEs == 1, int, float>::type sum = 0;
    for (uint32_t k = 0; k < red; k++)
      sum += element<E>(p + (kTransP ? (int64_t)k * a.p_stride : (int64_t)k * E::kEs)) *
             element<E>(q + (kTransQ ? (int64_t)k * a.q_stride : (int64_t)k * E::kEs));
    float v = (float)sum;
    if constexpr (E::kEs == 1) {
      v = scaled(v, a.row_scale[row] * a.col_scale[col], a.bias != nullptr, a.bias ? a.bias[col] : 0.f);
    }
    ((typename D::bits*)a.out)[out + (int64_t)row * a.out_stride + col] = D::from_f32(v);
  }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// A few rows against a matrix: what counts is that the matrix streams.  A workgroup of 8 waves takes 16 columns and
// each wave every eighth 128-byte line of k.  A load brings 8 rows of one line, whole lines and not kept in the caches:
// read by itself a 235 MB matrix comes in at 6.1 TB/s that way, at 4.1 to 5.3 TB/s where an instruction reads 64 bytes of
// each of 16 rows as the matrix instructions want them.  A corner of LDS that is the wave's own turns one layout into the
// other, without a barrier.  The eight partial sums are added up in LDS in the waves' order.
// With SX the rows come as floating-point numbers and are converted to 8 bits in the workgroup, into LDS, while the first
// lines of the matrix are on their way: one launch instead of two.
// MT blocks of 16 rows share what is read of the matrix.
constexpr int kFewCols = 16, kFewWaves = 8, kFewThreads = kFewWaves * 64;
constexpr int kFewConverted = 16;    // rows that are converted here at most: every 16 columns read them again
constexpr int kFewTogether = 4;      // rows up to which the whole workgroup converts each of them
constexpr uint32_t kFewLds = 32768;  // bytes of converted rows at most

struct FewArgs {
  MatmulArgs m;
  const void* x;     // SX: rows to be converted
  int64_t x_stride;  // elements
};

template <typename E, uint32_t KIND, typename D, typename SX, int MT>
__global__ __launch_bounds__(kFewThreads) void etha_few_rows_kernel(const FewArgs few) {
  constexpr bool kConvert = !std::is_void_v<SX>;
  constexpr int kRows = MT * 16, kAhead = MT == 1 ? 4 : 2;
  typedef typename std::conditional<E::kEs == 1, int, float>::type sum_t;
  const MatmulArgs& a = few.m;
  // a line of 16 columns and of the rows, later the sums; all of it the wave's own until the last barrier
  __shared__ __align__(1024) char s_turn[kFewWaves][2048 + (kConvert ? 0 : MT * 2048)];
  __shared__ __align__(16) char s_x[kConvert ? kFewLds + kFewConverted * 32 : 16];
  __shared__ uint32_t s_top[kConvert ? kFewConverted : 1][kFewWaves];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col_tiles = (a.cols + kFewCols - 1) / kFewCols;
  const uint32_t col0 = blockIdx.x % col_tiles * kFewCols, row_id = blockIdx.x / col_tiles;
  uint32_t row0 = row_id * kRows, row_end = a.rows, red = a.red;
  const char *p = a.p, *q = a.q;
  if constexpr (KIND != kPlain) {
    const GroupTile g = find_tile<kRows>(a, row_id);
    if (!g.found) return;
    row0 = g.lo + g.tile * kRows;
    row_end = g.hi;
    if (g.group == a.n_groups) red = 0;
    else q += (int64_t)g.group * a.q_group_stride;
  }
  const uint32_t n_rows = row_end - row0 < kRows ? row_end - row0 : kRows;
  const int64_t bytes = (int64_t)red * E::kEs;
  const uint32_t whole = (uint32_t)(bytes / 128);
  // a load: row lane >> 3 of 8, piece lane & 7 of its line; columns past the last repeat it, rows past the last are not read
  const uint32_t lrow = lane >> 3, at = (lane & 7) * 16;
  const char *wp[2], *xp[2 * MT];
  #pragma unroll
  for (int j = 0; j < 2; j++) {
    const uint32_t c = col0 + j * 8 + lrow;
    wp[j] = q + (int64_t)(c < a.cols ? c : a.cols - 1) * a.q_stride + at;
  }
  #pragma unroll
  for (int j = 0; j < 2 * MT; j++) xp[j] = p + (int64_t)(row0 + j * 8 + lrow) * a.p_stride + at;
  char* turn = s_turn[wave];
  const uint32_t put = lrow * 128 + (((lane & 7) ^ lrow) << 4);
  const uint32_t r = lane & 15, pitch = (uint32_t)(bytes + 127) / 128 * 128 + 32;  // of converted rows
  typename E::acc acc[MT] = {};
  u32x4 w[kAhead][2], x[kAhead][2 * MT] = {};
  const auto load = [&](uint32_t line) {
    #pragma unroll
    for (int u = 0; u < kAhead; u++) {
      const int64_t k = (int64_t)(line + u * kFewWaves) * 128;
      #pragma unroll
      for (int j = 0; j < 2; j++) w[u][j] = load_raw<16, true>(wp[j] + k);
      if constexpr (!kConvert) {
        #pragma unroll
        for (int j = 0; j < 2 * MT; j++)
          if (j * 8 + lrow < n_rows) x[u][j] = load_raw<16>(xp[j] + k);
      }
    }
  };
  const auto multiply = [&](int u, uint32_t line) {
    #pragma unroll
    for (int j = 0; j < 2; j++) *(u32x4*)(turn + j * 1024 + put) = w[u][j];
    if constexpr (!kConvert) {
      #pragma unroll
      for (int j = 0; j < 2 * MT; j++)
        if (j * 8 < n_rows) *(u32x4*)(turn + 2048 + j * 1024 + put) = x[u][j];
    }
    #pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t piece = h * 4 + (lane >> 4), get = r * 128 + ((piece ^ (r & 7)) << 4);
      const u32x4 fw = *(const u32x4*)(turn + get);
      #pragma unroll
      for (int m = 0; m < MT; m++) {
        if (m * 16 >= n_rows) break;
        const uint32_t xr = m * 16 + r < n_rows ? m * 16 + r : n_rows - 1;  // rows past the last repeat it, and are dropped
        u32x4 fx;
        if constexpr (kConvert) fx = *(const u32x4*)(s_x + xr * pitch + line * 128 + piece * 16);
        else fx = *(const u32x4*)(turn + 2048 + xr * 128 + ((piece ^ (xr & 7)) << 4));
        acc[m] = E::mfma(fw, fx, acc[m]);
      }
    }
  };
  // lines wave, wave + 8, ...: batches of kAhead of them, then one by one
  uint32_t line = wave;
  const auto batch = [&]() { return line + (kAhead - 1) * kFewWaves < whole; };
  const bool early = batch();
  if (early) load(line);
  if constexpr (kConvert) {
    const typename SX::bits* rows = (const typename SX::bits*)few.x;
    if (n_rows <= kFewTogether) {
      const uint32_t k0 = threadIdx.x * 8;
      float kept[kFewTogether][8];  // the first 4096 of a row stay in registers, all rows' loads are on their way at once
      #pragma unroll
      for (uint32_t m = 0; m < kFewTogether; m++)
        if (m < n_rows) load_f32<SX, 8>(kept[m], rows + (int64_t)(row0 + m) * few.x_stride + k0, (int64_t)red - k0);
      #pragma unroll
      for (uint32_t m = 0; m < kFewTogether; m++)
        if (m < n_rows) {
          uint32_t top = largest_bits(kept[m], 0);
          for (uint32_t k = k0 + kFewThreads * 8; k < red; k += kFewThreads * 8) {
            float v[8];
            load_f32<SX, 8>(v, rows + (int64_t)(row0 + m) * few.x_stride + k, (int64_t)red - k);
            top = largest_bits(v, top);
          }
          top = group_max<64>(top);
          if (lane == 0) s_top[m][wave] = top;
        }
      __syncthreads();
      #pragma unroll
      for (uint32_t m = 0; m < kFewTogether; m++)
        if (m < n_rows) {
          uint32_t top = 0;
          #pragma unroll
          for (int i = 0; i < kFewWaves; i++) top = s_top[m][i] > top ? s_top[m][i] : top;
          const RowScale scale(top);
          if (k0 < pitch - 32) *(u32x2*)(s_x + m * pitch + k0) = scale.pack<SX>(kept[m]);  // past the end of k: zeros
          for (uint32_t k = k0 + kFewThreads * 8; k < pitch - 32; k += kFewThreads * 8) {
            float v[8];
            load_f32<SX, 8>(v, rows + (int64_t)(row0 + m) * few.x_stride + k, (int64_t)red - k);
            *(u32x2*)(s_x + m * pitch + k) = scale.pack<SX>(v);
          }
        }
    } else {
      for (uint32_t m = wave; m < n_rows; m += kFewWaves) {  // a wave a row, which is read twice
        const typename SX::bits* x = rows + (int64_t)(row0 + m) * few.x_stride;
        uint32_t top = 0;
        #pragma unroll 4
        for (uint32_t k = lane * 8; k < red; k += 64 * 8) {
          float v[8];
          load_f32<SX, 8>(v, x + k, (int64_t)red - k);
          top = largest_bits(v, top);
        }
        top = group_max<64>(top);
        if (lane < kFewWaves) s_top[m][lane] = top;
        const RowScale scale(top);
        for (uint32_t k = lane * 8; k < pitch - 32; k += 64 * 8) {
          float v[8];
          load_f32<SX, 8>(v, x + k, (int64_t)red - k);
          *(u32x2*)(s_x + m * pitch + k) = scale.pack<SX>(v);
        }
      }
    }
    __syncthreads();
  }
  if (early) {
    for (;;) {
      #pragma unroll
      for (int u = 0; u < kAhead; u++) multiply(u, line + u * kFewWaves);
      line += kAhead * kFewWaves;
      if (!batch()) break;
      load(line);
    }
  }
  for (; line * 128 < bytes; line += kFewWaves) {
    #pragma unroll
    for (int j = 0; j < 2; j++) {
      const int64_t k = (int64_t)line * 128, left = bytes - k - at;
      w[0][j] = load_part<E::kEs>(wp[j] + k, left);
    }
    if constexpr (!kConvert) {
      #pragma unroll
      for (int j = 0; j < 2 * MT; j++) {
        const int64_t k = (int64_t)line * 128, left = bytes - k - at;
        if (j * 8 + lrow < n_rows) x[0][j] = load_part<E::kEs>(xp[j] + k, left);
      }
    }
    multiply(0, line);
  }
  sum_t* sums = (sum_t*)turn;
  #pragma unroll
  for (int m = 0; m < MT; m++)
    #pragma unroll
    for (int c = 0; c < 4; c++) sums[m * 256 + lane * 4 + c] = acc[m][c];
  __syncthreads();
  #pragma unroll
  for (int e = 0; e < (MT + 1) / 2; e++) {
    const uint32_t t = threadIdx.x + e * kFewThreads;
    const uint32_t row = row0 + (t >> 8) * 16 + (t >> 2 & 15), col = col0 + (t >> 6 & 3) * 4 + (t & 3);
    if (t >= kRows * kFewCols || row >= row_end || col >= a.cols) continue;
    sum_t sum = ((const sum_t*)s_turn[0])[t];
    #pragma unroll
    for (int i = 1; i < kFewWaves; i++) sum += ((const sum_t*)s_turn[i])[t];
    float v = (float)sum;
    if constexpr (E::kEs == 1) {
      float row_scale;
      if constexpr (kConvert) {
        uint32_t top = 0;
        #pragma unroll
        for (int i = 0; i < kFewWaves; i++) top = s_top[row - row0][i] > top ? s_top[row - row0][i] : top;
        row_scale = RowScale(top).scale;
      } else {
        row_scale = a.row_scale[row];
      }
      v = scaled(v, row_scale * a.col_scale[col], a.bias != nullptr, a.bias ? a.bias[col] : 0.f);
    }
    ((typename D::bits*)a.out)[(int64_t)row * a.out_stride + col] = D::from_f32(v);
  }
}

// A few rows against matrices that lie transposed (the gradient of the rows): the same stream.  A workgroup takes 64 columns,
// which are 128 bytes of a row of memory, and each wave every eighth run of 64 rows of k; the transposing LDS load turns
// them.  Pieces that reach over the end of a row or of k are handled as RegisterStage does it.
constexpr int kFewColsT = 64;

template <typename E, typename D>
__global__ __launch_bounds__(kFewThreads) void etha_few_rows_transposed_kernel(const MatmulArgs a) {
  typedef Operand<E, true, kFewColsT, 128> OpQ;  // for the layouts of the LDS tiles
  typedef Operand<E, false, 16, 128> OpP;
  constexpr uint32_t kRun = 64;
  __shared__ __align__(1024) char s_tile[kFewWaves][OpQ::kBytes + OpP::kBytes];  // the wave's own until the last barrier
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t col_tiles = (a.cols + kFewColsT - 1) / kFewColsT;
  const uint32_t col0 = blockIdx.x % col_tiles * kFewColsT;
  const GroupTile g = find_tile<16>(a, blockIdx.x / col_tiles);
  if (!g.found) return;
  const uint32_t row0 = g.lo + g.tile * 16, n_rows = g.hi - row0 < 16 ? g.hi - row0 : 16;
  const uint32_t n_cols = a.cols - col0 < kFewColsT ? a.cols - col0 : kFewColsT;
  const uint32_t red = g.group == a.n_groups ? 0 : a.red;
  const char* q = a.q + (g.group == a.n_groups ? 0 : (int64_t)g.group * a.q_group_stride) + (int64_t)col0 * 2;
  const char* p = a.p + (int64_t)row0 * a.p_stride;
  char* tile = s_tile[wave];
  const uint32_t row = lane >> 3, piece = (lane & 7) * 16;  // of 8 rows of 128 bytes, in memory
  const int left_q = (int)(n_cols * 2) - (int)piece;
  const int at_q = left_q >= 16 ? (int)piece : (int)(n_cols * 2) - 16;
  const uint32_t shift_q = left_q >= 16 || left_q <= 0 ? 0 : 16 - left_q;
  const uint32_t prow[2] = {row < n_rows ? row : n_rows - 1, row + 8 < n_rows ? row + 8 : n_rows - 1};
  f32x4 acc[4] = {};
  for (uint32_t k0 = wave * kRun; k0 < red; k0 += kFewWaves * kRun) {
    const uint32_t inside = red - k0 < kRun ? red - k0 : kRun;
    const int left_p = (int)((red - k0) * 2) - (int)piece;
    const uint32_t at_p = left_p >= 16 ? k0 * 2 + piece : red * 2 - 16;
    const uint32_t shift_p = left_p >= 16 ? 0 : left_p > 0 ? 16 - left_p : 16;
    u32x4 vq[8], vp[2];
    #pragma unroll
    for (uint32_t i = 0; i < 8; i++)
      vq[i] = load_raw<16, true>(q + (int64_t)(k0 + (i * 8 + row < inside ? i * 8 + row : inside - 1)) * a.q_stride + at_q);
    #pragma unroll
    for (int i = 0; i < 2; i++) vp[i] = load_raw<16>(p + (int64_t)prow[i] * a.p_stride + at_p);
    if (inside < kRun || n_cols < kFewColsT) {
      #pragma unroll
      for (uint32_t i = 0; i < 8; i++) vq[i] = shift_bytes(vq[i], i * 8 + row >= inside ? 16 : shift_q);
      #pragma unroll
      for (int i = 0; i < 2; i++) vp[i] = shift_bytes(vp[i], shift_p);
    }
    #pragma unroll
    for (uint32_t i = 0; i < 8; i++) *(u32x4*)(tile + (i * 8 + row) * 128 + OpQ::swizzle(i * 8 + row, lane & 7) * 16) = vq[i];
    #pragma unroll
    for (uint32_t i = 0; i < 2; i++) *(u32x4*)(tile + OpQ::kBytes + (i * 8 + row) * 128 + OpP::swizzle(i * 8 + row, lane & 7) * 16) = vp[i];
    #pragma unroll
    for (int h = 0; h < 2; h++) {
      const u32x4 fp = OpP::fragment(tile + OpQ::kBytes, 0, h * 4);
      #pragma unroll
      for (int j = 0; j < 4; j++) acc[j] = E::mfma(OpQ::fragment(tile, j * 16, h * 4), fp, acc[j]);
    }
  }
  float* sums = (float*)tile;
  #pragma unroll
  for (int j = 0; j < 4; j++)
    #pragma unroll
    for (int c = 0; c < 4; c++) sums[j * 256 + lane * 4 + c] = acc[j][c];
  __syncthreads();
  #pragma unroll
  for (int e = 0; e < 2; e++) {
    const uint32_t t = threadIdx.x + e * kFewThreads;
    const uint32_t out_row = row0 + (t >> 2 & 15), col = col0 + (t >> 8) * 16 + (t >> 6 & 3) * 4 + (t & 3);
    if (out_row >= g.hi || col >= a.cols) continue;
    float sum = ((const float*)s_tile[0])[t];
    #pragma unroll
    for (int i = 1; i < kFewWaves; i++) sum += ((const float*)s_tile[i])[t];
    ((typename D::bits*)a.out)[(int64_t)out_row * a.out_stride + col] = D::from_f32(sum);
  }
}

// The parts of a sum over a group's rows, added up in their order; four columns a work-item.
template <typename D>
__global__ __launch_bounds__(256) void etha_join_parts_kernel(const float* parts, uint32_t splits, int64_t split_stride, uint64_t rows,
                                                              uint32_t group_rows, uint32_t cols, typename D::bits* out, int64_t out_stride,
                                                              int64_t out_group_stride) {
  const uint32_t vecs = (cols + 3) / 4;
  for (uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x; id < rows * vecs; id += (uint64_t)gridDim.x * 256) {
    const uint64_t row = id / vecs;
    const uint32_t col = (uint32_t)(id % vecs) * 4;
    const int64_t left = (int64_t)cols - col;
    float sum[4] = {}, v[4];
    #pragma unroll 4
    for (uint32_t s = 0; s < splits; s++) {
      load_f32<F32, 4>(v, (const uint32_t*)parts + s * split_stride + (int64_t)row * cols + col, left);
      #pragma unroll
      for (int i = 0; i < 4; i++) sum[i] += v[i];
    }
    store_f32<D, 4>(out + (int64_t)(row / group_rows) * out_group_stride + (int64_t)(row % group_rows) * out_stride + col, sum, left);
  }
}

int launched(const char* name) {
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(ETHA_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
  return ETHA_OK;
}

int check_sizes(const char* what, uint64_t rows, uint64_t cols, uint64_t red, uint64_t most_red) {
  if (rows >= 1ull << 31 || cols >= 1ull << 31)
    return fail(ETHA_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows and columns", what);
  if (red > most_red) return fail(ETHA_ERR_UNSUPPORTED, "%s: a sum over %llu elements; at most %llu", what, (unsigned long long)red,
                                  (unsigned long long)most_red);
  return ETHA_OK;
}

// Whether an operand's tiles can be brought straight into LDS, see DirectStage.  `across`: elements of a row of memory
// where it lies transposed; rows that overlap (a broadcast gradient) would leave what is past the end of k within the tile.
constexpr uint32_t kMostStride = 1u << 23;  // bytes between rows: offsets within a tile of 256 of them have 32 bits

bool is_direct(const void* base, int64_t stride, int64_t group_stride, uint64_t k_bytes, bool trans, uint64_t across) {
  return !(((uintptr_t)base | (uint64_t)stride | (uint64_t)group_stride) & 15) && stride >= 0 && stride < 1 << 22 &&
         (trans ? (uint64_t)stride >= across * 2 : !(k_bytes & 15));
}

// Tile shapes.  Measured on grouped bf16 products, 8 x [3584, 4096]: 256 x 256 with 8 waves 433 us at 16384 rows (4 waves
// 600 us, stages of 64 bytes of k 465 us), 128 x 128 with 8 waves 59 us at 1024 rows (4 waves 87 us), 32 x 64 52 us at 256.
typedef Shape<256, 256, 2, 4, 2> ShapeL;
typedef Shape<128, 128, 2, 4, 2> ShapeM;  // also for operands that go through registers
typedef Shape<32, 64, 1, 4, 6> ShapeS;

// No group wastes more than one row tile, and a group with rows has at least one.
uint64_t row_tiles_of(const MatmulArgs& a, uint32_t kind, int bm) {
  if (kind == kPlain) return ((uint64_t)a.rows + bm - 1) / bm;
  if (kind == kGroupReduce) return ((uint64_t)a.rows + bm - 1) / bm * a.n_groups;
  const uint64_t groups = (uint64_t)a.n_groups + 2 < a.rows ? a.n_groups + 2 : a.rows;
  return (a.rows - groups) / bm + groups;
}

// Workgroups of a launch: with 512 work-items each, half of what a grid may have.
constexpr uint64_t kMostBlocks = 1u << 22;

template <typename E, uint32_t KIND, typename D, typename S, template <typename> class STAGE>
int launch_matmul(const char* what, const MatmulArgs& a, void* stream) {
  const uint64_t row_tiles = row_tiles_of(a, KIND, S::BM);
  const uint64_t col_tiles = ((uint64_t)a.cols + S::BN - 1) / S::BN, blocks = row_tiles * col_tiles;
  if (blocks >= kMostBlocks) return fail(ETHA_ERR_UNSUPPORTED, "%s: the product is too large for one call", what);
  if (!blocks) return ETHA_OK;
  hipLaunchKernelGGL((etha_matmul_kernel<E, KIND, D, S, STAGE>), dim3((uint32_t)blocks, a.splits > 1 ? a.splits : 1), dim3(S::kThreads), 0, (hipStream_t)stream, a);
  return launched("etha_matmul_kernel");
}

template <typename E, uint32_t KIND, typename D, typename S>
int launch_shape(const char* what, const MatmulArgs& a, bool direct, void* stream) {
  return direct ? launch_matmul<E, KIND, D, S, DirectStage>(what, a, stream) : launch_matmul<E, KIND, D, S, RegisterStage>(what, a, stream);
}

template <typename E, uint32_t KIND, typename D, typename SX, int MT>
int launch_few(const char* what, const FewArgs& few, void* stream) {
  const uint64_t blocks = row_tiles_of(few.m, KIND, MT * 16) * (((uint64_t)few.m.cols + kFewCols - 1) / kFewCols);
  if (blocks >= kMostBlocks) return fail(ETHA_ERR_UNSUPPORTED, "%s: the product is too large for one call", what);
  hipLaunchKernelGGL((etha_few_rows_kernel<E, KIND, D, SX, MT>), dim3((uint32_t)blocks), dim3(kFewThreads), 0, (hipStream_t)stream, few);
  return launched("etha_few_rows_kernel");
}

// What a choice of tiles costs, in microseconds, by what bounded the shapes where they were measured: a workgroup takes in
// its operands at about 45 GB/s and needs `fixed` to begin and to write its results, all of them together take in `tbs`, and
// the matrices come from memory at `gbs`.  A rule on sizes alone; the rows of a group are taken as even, half a tile a group
// as lost.
struct TileCost {
  int bm, bn, resident;
  double fixed, tbs, gbs;
};
double tile_cost(const MatmulArgs& a, uint32_t kind, int es, const TileCost& t) {
  const double k_bytes = (double)a.red * es;
  const double groups = kind == kPlain ? 1 : a.n_groups < a.rows ? (a.n_groups ? a.n_groups : 1) : a.rows;
  const double high = a.rows / groups < t.bm ? a.rows / groups : t.bm;  // rows of a tile that there are
  double row_tiles = kind == kPlain ? (double)((a.rows + t.bm - 1) / t.bm) : a.rows / (double)t.bm + groups / 2;
  if (row_tiles < groups) row_tiles = groups;
  const double tiles = row_tiles * ((a.cols + t.bn - 1) / t.bn), bytes = (high + t.bn) * k_bytes;
  const double rounds = (double)(uint64_t)((tiles + t.resident - 1) / t.resident);
  double us = rounds * (bytes / 45e3 + t.fixed);
  if (tiles * bytes / t.tbs / 1e6 + t.fixed > us) us = tiles * bytes / t.tbs / 1e6 + t.fixed;
  if (groups * a.cols * k_bytes / t.gbs / 1e3 > us) us = groups * a.cols * k_bytes / t.gbs / 1e3;
  return us;
}

// The kernel that a product takes (ETHA_PRODUCT_*).
uint32_t choose_kernel(const MatmulArgs& a, uint32_t kind, int es, bool direct) {
  const uint64_t p_row = (uint64_t)(kind == kGroupReduce ? a.rows : a.red) * es;
  const uint64_t q_row = (uint64_t)(kind == kGroupReduce || kind == kGroupRowsT ? a.cols : a.red) * es;
  if (!direct && (p_row < 16 || q_row < 16)) return ETHA_PRODUCT_SHORT;
  if (kind == kGroupReduce) {
    // the large tile wherever there are enough of them for every CU, also for few rows, where all there is to do is writing
    // the results (16 rows, 8 x [3584, 4096]: 53 us, 63 us with the middle one)
    const uint64_t tiles = row_tiles_of(a, kind, ShapeL::BM) * (((uint64_t)a.cols + ShapeL::BN - 1) / ShapeL::BN);
    return a.splits < 2 && tiles >= 192 ? ETHA_PRODUCT_TILE_256 : ETHA_PRODUCT_TILE_128;
  }
  const double none = 1e30;
  const bool few = kind != kGroupRowsT;
  const TileCost shapes[6] = {
      few ? TileCost{16, kFewCols, 512, 2, 11, 6000} : TileCost{16, kFewColsT, 512, 2, 7, 6000},
      {32, kFewCols, 512, 2, 11, 6000},
      {64, kFewCols, 256, 2, 11, 6000},
      {ShapeS::BM, ShapeS::BN, 512, 3, 11, 4600},
      {ShapeM::BM, ShapeM::BN, 512, 4, 11, 5200},
      {ShapeL::BM, ShapeL::BN, 256, 8, 11, 4600},
  };
  static const uint32_t kernels[6] = {ETHA_PRODUCT_FEW_16, ETHA_PRODUCT_FEW_32, ETHA_PRODUCT_FEW_64,
                                      ETHA_PRODUCT_TILE_32, ETHA_PRODUCT_TILE_128, ETHA_PRODUCT_TILE_256};
  double cost[6];
  for (int i = 0; i < 6; i++) {
    cost[i] = tile_cost(a, kind, es, shapes[i]);
    if (row_tiles_of(a, kind, shapes[i].bm) * (((uint64_t)a.cols + shapes[i].bn - 1) / shapes[i].bn) >= kMostBlocks)
      cost[i] += none;  // more than a launch takes: only if no shape fits, which the launch then refuses
  }
  if (!few) cost[1] = cost[2] = 2 * none;
  if (!few && (p_row < 16 || q_row < 16)) cost[0] = 2 * none;  // its loads begin 16 bytes before the end of a row
  int best = 0;
  for (int i = 1; i < 6; i++)
    if (cost[i] < cost[best]) best = i;
  return kernels[best];
}

template <typename E, uint32_t KIND, typename D>
int shaped_matmul(const char* what, const MatmulArgs& a, bool direct, void* stream) {
  const uint32_t kernel = choose_kernel(a, KIND, E::kEs, direct);
  if (kernel == ETHA_PRODUCT_SHORT) {
    const uint64_t blocks = ((KIND == kGroupReduce ? a.n_groups : 1ull) * a.rows * a.cols + 255) / 256;
    hipLaunchKernelGGL((etha_matmul_short_kernel<E, KIND, D>), dim3((uint32_t)(blocks < 1u << 20 ? blocks : 1u << 20)), dim3(256), 0,
                       (hipStream_t)stream, a);
    return launched("etha_matmul_short_kernel");
  }
  if (kernel == ETHA_PRODUCT_TILE_256) return launch_shape<E, KIND, D, ShapeL>(what, a, direct, stream);
  if constexpr (KIND == kGroupReduce) {
    return launch_shape<E, KIND, D, ShapeM>(what, a, direct, stream);
  } else {
    if constexpr (KIND != kGroupRowsT) {
      FewArgs args = {};
      args.m = a;
      if (kernel == ETHA_PRODUCT_FEW_16) return launch_few<E, KIND, D, void, 1>(what, args, stream);
      if (kernel == ETHA_PRODUCT_FEW_32) return launch_few<E, KIND, D, void, 2>(what, args, stream);
      if (kernel == ETHA_PRODUCT_FEW_64) return launch_few<E, KIND, D, void, 4>(what, args, stream);
    } else {
      if (kernel == ETHA_PRODUCT_FEW_16) {
        const uint64_t blocks = row_tiles_of(a, KIND, 16) * (((uint64_t)a.cols + kFewColsT - 1) / kFewColsT);
        if (blocks >= kMostBlocks) return fail(ETHA_ERR_UNSUPPORTED, "%s: the product is too large for one call", what);
        hipLaunchKernelGGL((etha_few_rows_transposed_kernel<E, D>), dim3((uint32_t)blocks), dim3(kFewThreads), 0, (hipStream_t)stream, a);
        return launched("etha_few_rows_transposed_kernel");
      }
    }
    if (kernel == ETHA_PRODUCT_TILE_128) return launch_shape<E, KIND, D, ShapeM>(what, a, direct, stream);
    return launch_shape<E, KIND, D, ShapeS>(what, a, direct, stream);
  }
}

bool takes_direct(const MatmulArgs& a, uint32_t kind, int es) {
  const uint64_t k_bytes = (uint64_t)a.red * es;
  return is_direct(a.p, a.p_stride, 0, k_bytes, kind == kGroupReduce, a.rows) &&
         is_direct(a.q, a.q_stride, a.q_group_stride, k_bytes, kind == kGroupReduce || kind == kGroupRowsT, a.cols);
}

template <typename E, uint32_t KIND>
int run_matmul(const char* what, const MatmulArgs& a, uint32_t out_dtype, void* stream) {
  if (a.p_stride < 0 || a.q_stride < 0 || a.p_stride > kMostStride || a.q_stride > kMostStride)
    return fail(ETHA_ERR_UNSUPPORTED, "%s: rows have to lie at most %u bytes apart", what, kMostStride);
  const uint64_t k_bytes = (uint64_t)a.red * E::kEs;
  if (KIND != kGroupReduce && k_bytes > 1u << 30) return fail(ETHA_ERR_UNSUPPORTED, "%s: sums over at most 2^30 bytes of a row", what);
  const bool direct = takes_direct(a, KIND, E::kEs);
  if (out_dtype == ETHA_F32) return shaped_matmul<E, KIND, F32>(what, a, direct, stream);
  if (out_dtype == ETHA_BF16) return shaped_matmul<E, KIND, BF16>(what, a, direct, stream);
  return shaped_matmul<E, KIND, F16>(what, a, direct, stream);
}

bool is_out(uint32_t dtype) { return dtype == ETHA_F32 || dtype == ETHA_BF16 || dtype == ETHA_F16; }

// Rows that the few-rows kernel converts itself.  Every 16 columns convert them again while their part of the matrix
// arrives, which is less than a launch where that is little (16 x 2048 x 2048: 9.5 to 12.3 us, 13.6 us with a launch of its
// own; 8 x 4096 x 4096: 11.3 or 16.9 us, by how the workgroups come to lie on the CUs, 13.6 us) and the workgroups are all
// resident or the rows short (8 x 14336 x 1024: 10.2 to 12.9 us, 13.5 us; 4 x 14336 x 2048: 14.9 us, 13.5 us); a single row
// always is (14336 x 4096: 14.4 us, 16.5 us).
bool is_few(uint64_t rows, uint64_t cols, uint64_t width) {
  const uint64_t padded = (width + 127) / 128 * 128;
  if (rows > kFewConverted || rows * padded > kFewLds || (cols + kFewCols - 1) / kFewCols >= kMostBlocks) return false;
  return rows == 1 || (rows * padded * ((cols + 4095) / 4096) <= kFewLds && (cols <= 8192 || padded <= 1024) &&
                       (rows <= kFewTogether || padded <= 2048));
}
uint64_t padded_width(uint64_t width) { return (width + 15) / 16 * 16; }

// Parts that the sum over a group's rows is cut into where its tiles are too few for the chip: about two workgroups a CU,
// each with at least two stages of an even group's rows (groups are uneven, the longest one is what is waited for).
uint32_t reduce_splits(uint64_t rows, uint64_t n_groups, uint64_t out_rows, uint64_t out_cols) {
  if (!n_groups || !out_rows || !out_cols) return 1;
  const uint64_t tiles = n_groups * ((out_rows + ShapeM::BM - 1) / ShapeM::BM) * ((out_cols + ShapeM::BN - 1) / ShapeM::BN);
  const uint64_t stages = rows / n_groups / 64;
  if (tiles > 192 || stages < 4 || out_rows * 2 < 16 || out_cols * 2 < 16) return 1;
  const uint64_t by_tiles = (512 + tiles - 1) / tiles, by_stages = stages / 2;
  const uint64_t splits = by_tiles < by_stages ? by_tiles : by_stages;
  return (uint32_t)(splits < 64 ? splits : 64);
}

template <uint32_t KIND>
int run_grouped(const char* what, const MatmulArgs& a, uint32_t dtype, uint32_t out_dtype, void* stream) {
  return dtype == ETHA_BF16 ? run_matmul<ElemBF16, KIND>(what, a, out_dtype, stream) : run_matmul<ElemF16, KIND>(what, a, out_dtype, stream);
}

int check_groups(const char* what, const void* offsets, uint64_t n_groups, uint32_t dtype, uint32_t out_dtype) {
  if (dtype != ETHA_BF16 && dtype != ETHA_F16) return fail(ETHA_ERR_UNSUPPORTED, "%s: element types are bf16 and f16", what);
  if (!is_out(out_dtype)) return fail(ETHA_ERR_UNSUPPORTED, "%s: results are f32, bf16 or f16", what);
  if (n_groups > 1u << 16) return fail(ETHA_ERR_UNSUPPORTED, "%s: at most 65536 groups", what);
  if (!offsets) return fail(ETHA_ERR_INVALID, "%s: null offsets", what);
  return ETHA_OK;
}

}  // namespace

extern "C" {

int etha_int8_matmul(const int8_t* x, const float* x_scale, uint64_t rows, int64_t x_stride, const int8_t* w, const float* w_scale,
                     uint64_t cols, int64_t w_stride, uint64_t width, const float* bias, void* out, uint32_t out_dtype,
                     int64_t out_stride, void* stream) {
  const int rc = check_sizes("etha_int8_matmul", rows, cols, width, ETHA_INT8_MAX_WIDTH);
  if (rc != ETHA_OK) return rc;
  if (!is_out(out_dtype)) return fail(ETHA_ERR_UNSUPPORTED, "etha_int8_matmul: results are f32, bf16 or f16");
  if (!rows || !cols) return ETHA_OK;
  if ((width && (!x || !w)) || !x_scale || !w_scale || !out) return fail(ETHA_ERR_INVALID, "etha_int8_matmul: null tensor");
  MatmulArgs a = {};
  a.p = (const char*)x;
  a.q = (const char*)w;
  a.out = out;
  a.p_stride = x_stride;
  a.q_stride = w_stride;
  a.out_stride = out_stride;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.red = (uint32_t)width;
  a.row_scale = x_scale;
  a.col_scale = w_scale;
  a.bias = bias;
  return run_matmul<ElemI8, kPlain>("etha_int8_matmul", a, out_dtype, stream);
}

int etha_product_kernel(uint32_t product, uint32_t dtype, const void* p, int64_t p_stride, const void* q, int64_t q_stride,
                        int64_t q_group_stride, uint64_t rows, uint64_t cols, uint64_t red, uint64_t n_groups, uint32_t* kernel,
                        int* direct) {
  if (!kernel || !direct) return fail(ETHA_ERR_INVALID, "etha_product_kernel: null result");
  if (product > kGroupReduce || (product == kPlain ? dtype != ETHA_I8 : dtype != ETHA_BF16 && dtype != ETHA_F16))
    return fail(ETHA_ERR_INVALID, "etha_product_kernel: no such product");
  const int rc = check_sizes("etha_product_kernel", rows, cols, red, (1ull << 31) - 1);
  if (rc != ETHA_OK) return rc;
  if (n_groups > 1u << 16 || !rows || !cols) return fail(ETHA_ERR_INVALID, "etha_product_kernel: nothing is launched for these sizes");
  const int es = product == kPlain ? 1 : 2;
  MatmulArgs a = {};
  a.p = (const char*)p;
  a.q = (const char*)q;
  a.p_stride = p_stride * es;
  a.q_stride = q_stride * es;
  a.q_group_stride = q_group_stride * es;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.red = (uint32_t)red;
  a.n_groups = (uint32_t)n_groups;
  if (product == kGroupReduce) a.splits = reduce_splits(red, n_groups, rows, cols);
  *direct = takes_direct(a, product, es);
  *kernel = choose_kernel(a, product, es, *direct != 0);
  return ETHA_OK;
}

int etha_int8_linear_workspace(uint64_t rows, uint64_t cols, uint64_t width, uint64_t* bytes) {
  if (!bytes) return fail(ETHA_ERR_INVALID, "etha_int8_linear_workspace: null result");
  const int rc = check_sizes("etha_int8_linear_workspace", rows, cols, width, ETHA_INT8_MAX_WIDTH);
  if (rc != ETHA_OK) return rc;
  *bytes = is_few(rows, cols, width) ? 0 : rows * padded_width(width) + rows * 4;
  return ETHA_OK;
}

int etha_int8_linear(const void* x, uint32_t dtype, uint64_t rows, int64_t x_stride, const int8_t* w, const float* w_scale,
                     uint64_t cols, int64_t w_stride, uint64_t width, const float* bias, void* out, uint32_t out_dtype,
                     int64_t out_stride, void* workspace, uint64_t workspace_bytes, void* stream) {
  int rc = check_sizes("etha_int8_linear", rows, cols, width, ETHA_INT8_MAX_WIDTH);
  if (rc != ETHA_OK) return rc;
  if (!is_out(dtype) || !is_out(out_dtype)) return fail(ETHA_ERR_UNSUPPORTED, "etha_int8_linear: element types are f32, bf16 and f16");
  if (!rows || !cols) return ETHA_OK;
  if ((width && (!x || !w)) || !w_scale || !out) return fail(ETHA_ERR_INVALID, "etha_int8_linear: null tensor");
  if (is_few(rows, cols, width)) {
    FewArgs few = {};
    few.x = x;
    few.x_stride = x_stride;
    few.m.q = (const char*)w;
    few.m.out = out;
    few.m.q_stride = w_stride;
    few.m.out_stride = out_stride;
    few.m.rows = (uint32_t)rows;
    few.m.cols = (uint32_t)cols;
    few.m.red = (uint32_t)width;
    few.m.col_scale = w_scale;
    few.m.bias = bias;
    with_type(dtype, [&](auto s) {
      with_type(out_dtype, [&](auto d) {
        rc = launch_few<ElemI8, kPlain, decltype(d), decltype(s), 1>("etha_int8_linear", few, stream);
      });
    });
    return rc;
  }
  const uint64_t pitch = padded_width(width);
  if (!workspace || workspace_bytes < rows * pitch + rows * 4 || ((uintptr_t)workspace & 15))
    return fail(ETHA_ERR_INVALID, "etha_int8_linear: the workspace has to hold %llu bytes at a 16-byte address",
                (unsigned long long)(rows * pitch + rows * 4));
  int8_t* values = (int8_t*)workspace;
  float* scales = (float*)((char*)workspace + rows * pitch);
  rc = etha_quantize_rows(x, dtype, rows, width, x_stride, values, (int64_t)pitch, scales, stream);
  if (rc != ETHA_OK) return rc;
  return etha_int8_matmul(values, scales, rows, (int64_t)pitch, w, w_scale, cols, w_stride, width, bias, out, out_dtype, out_stride, stream);
}

int etha_grouped_matmul(const void* x, uint32_t dtype, uint64_t rows, int64_t x_stride, const void* w, uint64_t n_groups,
                        uint64_t cols, uint64_t red, int64_t w_stride, int64_t w_group_stride, int w_transposed,
                        const int32_t* offsets, void* out, uint32_t out_dtype, int64_t out_stride, int zero_rest, void* stream) {
  int rc = check_groups("etha_grouped_matmul", offsets, n_groups, dtype, out_dtype);
  if (rc == ETHA_OK) rc = check_sizes("etha_grouped_matmul", rows, cols, red, (1ull << 31) - 1);
  if (rc != ETHA_OK) return rc;
  if (!rows || !cols) return ETHA_OK;
  if (!out || (red && (!x || (n_groups && !w)))) return fail(ETHA_ERR_INVALID, "etha_grouped_matmul: null tensor");
  MatmulArgs a = {};
  a.p = (const char*)x;
  a.q = (const char*)w;
  a.out = out;
  a.p_stride = x_stride * 2;
  a.q_stride = w_stride * 2;
  a.q_group_stride = w_group_stride * 2;
  a.out_stride = out_stride;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.red = (uint32_t)red;
  a.offsets = offsets;
  a.n_groups = (uint32_t)n_groups;
  a.zero_rest = zero_rest != 0;
  return w_transposed ? run_grouped<kGroupRowsT>("etha_grouped_matmul", a, dtype, out_dtype, stream)
                      : run_grouped<kGroupRows>("etha_grouped_matmul", a, dtype, out_dtype, stream);
}

int etha_grouped_matmul_reduce_workspace(uint64_t rows, uint64_t n_groups, uint64_t out_rows, uint64_t out_cols, uint64_t* bytes) {
  if (!bytes) return fail(ETHA_ERR_INVALID, "etha_grouped_matmul_reduce_workspace: null result");
  const int rc = check_sizes("etha_grouped_matmul_reduce_workspace", out_rows, out_cols, rows, (1ull << 31) - 1);
  if (rc != ETHA_OK) return rc;
  const uint64_t splits = reduce_splits(rows, n_groups, out_rows, out_cols);
  *bytes = splits < 2 ? 0 : splits * n_groups * out_rows * out_cols * 4;
  return ETHA_OK;
}

int etha_grouped_matmul_reduce(const void* grad, const void* x, uint32_t dtype, uint64_t rows, int64_t grad_stride, int64_t x_stride,
                               uint64_t n_groups, uint64_t out_rows, uint64_t out_cols, const int32_t* offsets, void* out,
                               uint32_t out_dtype, int64_t out_stride, int64_t out_group_stride, void* workspace,
                               uint64_t workspace_bytes, void* stream) {
  int rc = check_groups("etha_grouped_matmul_reduce", offsets, n_groups, dtype, out_dtype);
  if (rc == ETHA_OK) rc = check_sizes("etha_grouped_matmul_reduce", out_rows, out_cols, rows, (1ull << 31) - 1);
  if (rc != ETHA_OK) return rc;
  if (!n_groups || !out_rows || !out_cols) return ETHA_OK;
  if (!out || (rows && (!grad || !x))) return fail(ETHA_ERR_INVALID, "etha_grouped_matmul_reduce: null tensor");
  MatmulArgs a = {};
  a.p = (const char*)grad;
  a.q = (const char*)x;
  a.out = out;
  a.p_stride = grad_stride * 2;
  a.q_stride = x_stride * 2;
  a.out_stride = out_stride;
  a.out_group_stride = out_group_stride;
  a.rows = (uint32_t)out_rows;
  a.cols = (uint32_t)out_cols;
  a.red = (uint32_t)rows;
  a.offsets = offsets;
  a.n_groups = (uint32_t)n_groups;
  const uint32_t splits = reduce_splits(rows, n_groups, out_rows, out_cols);
  if (splits < 2) return run_grouped<kGroupReduce>("etha_grouped_matmul_reduce", a, dtype, out_dtype, stream);
  const uint64_t elements = n_groups * out_rows * out_cols;
  if (!workspace || workspace_bytes < splits * elements * 4 || ((uintptr_t)workspace & 15))
    return fail(ETHA_ERR_INVALID, "etha_grouped_matmul_reduce: the workspace has to hold %llu bytes at a 16-byte address",
                (unsigned long long)(splits * elements * 4));
  a.out = workspace;
  a.out_stride = (int64_t)out_cols;
  a.out_group_stride = (int64_t)(out_rows * out_cols);
  a.splits = splits;
  a.split_stride = (int64_t)elements;
  rc = run_grouped<kGroupReduce>("etha_grouped_matmul_reduce", a, dtype, ETHA_F32, stream);
  if (rc != ETHA_OK) return rc;
  const uint64_t blocks = (n_groups * out_rows * ((out_cols + 3) / 4) + 255) / 256;
  with_type(out_dtype, [&](auto d) {
    typedef decltype(d) D;
    hipLaunchKernelGGL((etha_join_parts_kernel<D>), dim3((uint32_t)(blocks < 1u << 20 ? blocks : 1u << 20)), dim3(256), 0, (hipStream_t)stream,
                       (const float*)workspace, splits, (int64_t)elements, n_groups * out_rows, (uint32_t)out_rows, (uint32_t)out_cols,
                       (typename D::bits*)out, out_stride, out_group_stride);
  });
  return launched("etha_join_parts_kernel");
}

}  // extern "C"
