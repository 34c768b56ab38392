// Matrix products on local shards, MI355X (gfx950): 8-bit integers with scales, and products grouped by expert.
//
// One tile kernel serves every product here: an output tile out[r, c] = sum_k P(r, k) * Q(c, k), where either operand may
// lie k-contiguous in memory or transposed (k as the memory row).  Tiles of both operands are staged through LDS as rows
// of 128 bytes of k (64 elements of 16 bits, 128 of 8 bits) and go through the matrix units, which need 16 bytes of k a
// lane for either type, so both share one layout.  The eight 16-byte pieces of LDS row r are stored at piece ^ (r & 7):
// the 16 lanes that read the same piece of 16 rows then touch all banks.
#include <hip/hip_runtime.h>

#include <cstdint>

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

// ---- staging through registers: any stride, any alignment --------------------------------------------------------
constexpr int kStageBytes = 128;  // of k, a row

// 16 bytes at p of which `left` exist; the others read as zero
template <int ES>
__device__ inline u32x4 load_part(const char* p, int64_t left) {
  if (left >= 16) return load_raw<16>(p);
  u32x4 v = {0, 0, 0, 0};
  if (left <= 0) return v;
  if constexpr (ES == 2) {
    #pragma unroll
    for (int i = 0; i < 8; i++)
      if (2 * i < left) v[i >> 1] |= (uint32_t)*(const uint16_t*)(p + 2 * i) << (16 * (i & 1));
  } else {
    #pragma unroll
    for (int i = 0; i < 16; i++)
      if (i < left) v[i >> 2] |= (uint32_t)*(const uint8_t*)(p + i) << (8 * (i & 3));
  }
  return v;
}

__device__ inline uint32_t lds_at(uint32_t row, uint32_t piece) { return row * kStageBytes + ((piece ^ (row & 7)) << 4); }

// One operand's tile of ROWS rows, THREADS work-items.  `n_rows` rows exist from `base` on; k0 is in elements.
template <int ES, bool TRANS, int ROWS, int THREADS>
struct Stage {
  static constexpr int kPer = ROWS * 8 / THREADS;
  u32x4 v[kPer];

  __device__ void load(const char* base, int64_t stride, uint32_t n_rows, uint32_t k0, uint32_t red) {
    #pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t id = threadIdx.x + i * THREADS;
      if constexpr (!TRANS) {
        const uint32_t row = id >> 3, piece = id & 7;
        const int64_t at = (int64_t)k0 * ES + piece * 16;
        v[i] = load_part<ES>(base + (int64_t)row * stride + at, row < n_rows ? (int64_t)red * ES - at : 0);
      } else {  // memory row = k, 8 tile rows a piece
        constexpr uint32_t kPieces = ROWS / 8;
        const uint32_t k = id / kPieces, piece = id % kPieces;
        v[i] = load_part<ES>(base + (int64_t)(k0 + k) * stride + piece * 16, k0 + k < red ? ((int64_t)n_rows - piece * 8) * 2 : 0);
      }
    }
  }
  __device__ void store(char* lds) const {
    #pragma unroll
    for (int i = 0; i < kPer; i++) {
      const uint32_t id = threadIdx.x + i * THREADS;
      if constexpr (!TRANS) {
        *(u32x4*)(lds + lds_at(id >> 3, id & 7)) = v[i];
      } else {
        constexpr uint32_t kPieces = ROWS / 8;
        const uint32_t k = id / kPieces, piece = id % kPieces;
        #pragma unroll
        for (int j = 0; j < 8; j++)
          *(uint16_t*)(lds + lds_at(piece * 8 + j, k >> 3) + (k & 7) * 2) = (uint16_t)(v[i][j >> 1] >> (16 * (j & 1)));
      }
    }
  }
};

// ---- one element of the result -----------------------------------------------------------------------------------
template <typename E, typename D>
__device__ inline void store_four(const MatmulArgs& a, typename D::bits* out, uint32_t row, uint32_t col, uint32_t cols,
                                  typename E::acc acc) {
  float v[4];
  if constexpr (E::kEs == 1) {  // the integer sum is exact; one product of scales, as the definition has it
    const float rs = a.row_scale[row];
    #pragma unroll
    for (int i = 0; i < 4; i++) {
      v[i] = 0.f;
      if (col + i < cols) {
        v[i] = (float)acc[i] * (rs * a.col_scale[col + i]);
        if (a.bias) v[i] += a.bias[col + i];
      }
    }
  } else {
    #pragma unroll
    for (int i = 0; i < 4; i++) v[i] = acc[i];
  }
  if (col < cols) store_f32<D, 4>(out + (int64_t)row * a.out_stride + col, v, (int64_t)cols - col);
}

// ---- the tile kernel -----------------------------------------------------------------------------------------------
constexpr int kTile = 128;

template <typename E, uint32_t KIND, typename D>
__global__ __launch_bounds__(256) void etha_matmul_kernel(const MatmulArgs a) {
  constexpr bool kTransP = KIND == kGroupReduce, kTransQ = KIND == kGroupReduce || KIND == kGroupRowsT;
  constexpr uint32_t kStageK = kStageBytes / E::kEs;
  __shared__ __align__(16) char s_p[kTile * kStageBytes];
  __shared__ __align__(16) char s_q[kTile * kStageBytes];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col_tiles = (a.cols + kTile - 1) / kTile;
  const uint32_t tile_col = blockIdx.x % col_tiles, rest = blockIdx.x / col_tiles;
  const uint32_t col0 = tile_col * kTile;
  uint32_t row0, row_end, red = a.red;
  const char *p = a.p, *q = a.q;
  typename D::bits* out = (typename D::bits*)a.out;
  bool zero = false;
  if constexpr (KIND == kPlain) {
    row0 = rest * kTile;
    row_end = a.rows;
  } else if constexpr (KIND == kGroupReduce) {
    const uint32_t row_tiles = (a.rows + kTile - 1) / kTile, group = rest / row_tiles;
    uint32_t lo, hi;
    group_bounds(a, group, &lo, &hi);
    red = hi - lo;
    p += (int64_t)lo * a.p_stride;
    q += (int64_t)lo * a.q_stride;
    out += (int64_t)group * a.out_group_stride;
    row0 = rest % row_tiles * kTile;
    row_end = a.rows;
  } else {
    const GroupTile t = find_tile<kTile>(a, rest);
    if (!t.found) return;
    row0 = t.lo + t.tile * kTile;
    row_end = t.hi;
    zero = t.group == a.n_groups;
    if (!zero) q += (int64_t)t.group * a.q_group_stride;
  }
  const uint32_t n_rows = row_end - row0 < kTile ? row_end - row0 : kTile;
  const uint32_t n_cols = a.cols - col0 < kTile ? a.cols - col0 : kTile;
  p += kTransP ? (int64_t)row0 * E::kEs : (int64_t)row0 * a.p_stride;
  q += kTransQ ? (int64_t)col0 * E::kEs : (int64_t)col0 * a.q_stride;

  typename E::acc acc[4][4] = {};
  const uint32_t wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  if (!zero) {
    Stage<E::kEs, kTransP, kTile, 256> sp;
    Stage<E::kEs, kTransQ, kTile, 256> sq;
    if (red) {
      sp.load(p, a.p_stride, n_rows, 0, red);
      sq.load(q, a.q_stride, n_cols, 0, red);
    }
    for (uint32_t k0 = 0; k0 < red; k0 += kStageK) {
      __syncthreads();
      sp.store(s_p);
      sq.store(s_q);
      __syncthreads();
      if (k0 + kStageK < red) {
        sp.load(p, a.p_stride, n_rows, k0 + kStageK, red);
        sq.load(q, a.q_stride, n_cols, k0 + kStageK, red);
      }
      #pragma unroll
      for (int s = 0; s < 2; s++) {
        u32x4 fp[4], fq[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) {
          fp[i] = *(const u32x4*)(s_p + lds_at(wr + i * 16 + (lane & 15), s * 4 + (lane >> 4)));
          fq[i] = *(const u32x4*)(s_q + lds_at(wc + i * 16 + (lane & 15), s * 4 + (lane >> 4)));
        }
        #pragma unroll
        for (int i = 0; i < 4; i++)
          #pragma unroll
          for (int j = 0; j < 4; j++) acc[i][j] = E::mfma(fq[j], fp[i], acc[i][j]);
      }
    }
  }
  // a lane holds row (lane & 15) and four consecutive columns of each 16 x 16 block
  #pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t row = row0 + wr + i * 16 + (lane & 15);
    if (row >= row_end) continue;
    #pragma unroll
    for (int j = 0; j < 4; j++) store_four<E, D>(a, out, row, col0 + wc + j * 16 + (lane >> 4) * 4, a.cols, acc[i][j]);
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

template <typename E, uint32_t KIND>
int run_matmul(const char* what, const MatmulArgs& a, uint64_t row_tiles, uint32_t out_dtype, void* stream) {
  const uint64_t col_tiles = ((uint64_t)a.cols + kTile - 1) / kTile;
  const uint64_t blocks = row_tiles * col_tiles;
  if (blocks >= 1ull << 24) return fail(ETHA_ERR_UNSUPPORTED, "%s: the product is too large for one call", what);
  if (!blocks) return ETHA_OK;
  const dim3 grid((uint32_t)blocks), block(256);
  if (out_dtype == ETHA_F32) hipLaunchKernelGGL((etha_matmul_kernel<E, KIND, F32>), grid, block, 0, (hipStream_t)stream, a);
  else if (out_dtype == ETHA_BF16) hipLaunchKernelGGL((etha_matmul_kernel<E, KIND, BF16>), grid, block, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((etha_matmul_kernel<E, KIND, F16>), grid, block, 0, (hipStream_t)stream, a);
  return launched("etha_matmul_kernel");
}

bool is_out(uint32_t dtype) { return dtype == ETHA_F32 || dtype == ETHA_BF16 || dtype == ETHA_F16; }

template <uint32_t KIND>
int run_grouped(const char* what, const MatmulArgs& a, uint64_t row_tiles, uint32_t dtype, uint32_t out_dtype, void* stream) {
  return dtype == ETHA_BF16 ? run_matmul<ElemBF16, KIND>(what, a, row_tiles, out_dtype, stream)
                            : run_matmul<ElemF16, KIND>(what, a, row_tiles, out_dtype, stream);
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
  return run_matmul<ElemI8, kPlain>("etha_int8_matmul", a, (rows + kTile - 1) / kTile, out_dtype, stream);
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
  // no group wastes more than one tile, and a group with rows has at least one
  const uint64_t groups = n_groups + 2 < rows ? n_groups + 2 : rows;
  const uint64_t tiles = (rows - groups) / kTile + groups;
  return w_transposed ? run_grouped<kGroupRowsT>("etha_grouped_matmul", a, tiles, dtype, out_dtype, stream)
                      : run_grouped<kGroupRows>("etha_grouped_matmul", a, tiles, dtype, out_dtype, stream);
}

int etha_grouped_matmul_reduce(const void* grad, const void* x, uint32_t dtype, uint64_t rows, int64_t grad_stride, int64_t x_stride,
                               uint64_t n_groups, uint64_t out_rows, uint64_t out_cols, const int32_t* offsets, void* out,
                               uint32_t out_dtype, int64_t out_stride, int64_t out_group_stride, void* stream) {
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
  const uint64_t tiles = (out_rows + kTile - 1) / kTile * n_groups;
  return run_grouped<kGroupReduce>("etha_grouped_matmul_reduce", a, tiles, dtype, out_dtype, stream);
}

}  // extern "C"
