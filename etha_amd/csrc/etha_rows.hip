// Row operators on local shards, MI355X (gfx950): embedding lookup, its gradient, conversion of rows to 8 bits.
//
// All three are bound by HBM: every element is read once and written once, and the arithmetic in between is a few
// operations.  Sums are held in fp32, one rounding at the end.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "etha_device.h"
#include "etha_internal.h"
#include "etha_reshard.h"

using etha_internal::fail;
using etha_internal::g_kernel_launches;
using namespace etha_device;

namespace {

constexpr int kWave = 64;

int launched(const char* name) {
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(ETHA_ERR_HIP, "%s: %s", name, hipGetErrorString(e));
  return ETHA_OK;
}

// Row of the shard that token i names, or `n_rows` where it is another shard's.
__device__ inline uint32_t local_row(const void* tokens, int wide, uint64_t i, int64_t first, uint32_t n_rows) {
  const int64_t id = wide ? ((const int64_t*)tokens)[i] : (int64_t)((const int32_t*)tokens)[i];
  // unsigned differences: an id far below `first` must not wrap into the shard
  return id >= first && (uint64_t)id - (uint64_t)first < n_rows ? (uint32_t)((uint64_t)id - (uint64_t)first) : n_rows;
}

// ---- embedding lookup ------------------------------------------------------------------------------------------
// y[t,:] = scale * W[row(t),:], zeros where the token is another shard's.  A work-item moves one vector; `lanes`
// work-items (a power of two) walk one row, so that narrow rows share a workgroup.
struct LookupArgs {
  const void* tokens;
  const void* weight;
  void* out;
  uint64_t n_tokens, width;
  int64_t first, weight_stride, out_stride;
  uint32_t n_rows, lanes_log2, wide;
  float scale;
};

// Elements of a work-item: 16 bytes of the narrower type (fp32 rows read as bf16, 16381 tokens of 4096: 20.0 us; 29.7 us
// with 16 bytes of the wider one).
constexpr int lookup_vec(int es, int eo) { return 16 / (es < eo ? es : eo); }

template <typename S, typename D>
__global__ __launch_bounds__(256) void etha_embedding_kernel(const LookupArgs a) {
  constexpr int N = lookup_vec(sizeof(typename S::bits), sizeof(typename D::bits));
  const uint32_t sub = threadIdx.x >> a.lanes_log2, lane = threadIdx.x & ((1u << a.lanes_log2) - 1);
  const uint32_t per_block = blockDim.x >> a.lanes_log2;
  const uint64_t col = ((uint64_t)blockIdx.y << a.lanes_log2 | lane) * N;
  if (col >= a.width) return;
  const int64_t left = (int64_t)(a.width - col);
  for (uint64_t t = (uint64_t)blockIdx.x * per_block + sub; t < a.n_tokens; t += (uint64_t)gridDim.x * per_block) {
    const uint32_t row = local_row(a.tokens, a.wide, t, a.first, a.n_rows);
    float v[N];
    if (row < a.n_rows) {
      load_f32<S, N>(v, (const typename S::bits*)a.weight + (int64_t)row * a.weight_stride + col, left);
      #pragma unroll
      for (int i = 0; i < N; i++) v[i] *= a.scale;
    } else {
      #pragma unroll
      for (int i = 0; i < N; i++) v[i] = 0.f;
    }
    store_f32<D, N, true>((typename D::bits*)a.out + (int64_t)t * a.out_stride + col, v, left);
  }
}

// ---- sorting tokens by row ---------------------------------------------------------------------------------------
// Tokens row by row, a row's positions in their own order, so that the sums that follow do not depend on timing.  One launch:
// a workgroup owns every 2^groups_log2-th row (frequent tokens lie close together) and looks through all tokens, a wave
// through a run of them.  It counts those of each of its rows, wave by wave, and those of the workgroups before it, which
// says where its own begin, and notes which they are; then every wave puts its tokens where the counts say.  Lanes whose
// tokens have the same row find each other with one ballot per bit.  57984 tokens of 21716 rows 22 us, 6965 of 6676 rows 7 us
// (a radix sort of two passes, with four launches, took 29 us and the gaps between them; one in a single workgroup 17 us for
// the latter; runs of rows instead of every 256th, with the tokens looked through twice, 57 us for the former).  The looking,
// some 10 instructions for 64 tokens, would take about 4 of those 22 us; how the rest is shared by clearing, scans and placing
// has not been measured.
constexpr uint32_t kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kSortNoted = 1024;
constexpr int kSortBinsLog2 = 10;
constexpr int kSortGroupsLog2 = 8;

// Exclusive sum over the workgroup's work-items and the sum of all; `sums` holds one word per wave.
__device__ inline uint32_t scan_block(uint32_t v, uint32_t* sums, uint32_t* all) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = v;
  #pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(inc, d);
    if (lane >= (uint32_t)d) inc += o;
  }
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  uint32_t base = 0, total = 0;
  #pragma unroll
  for (uint32_t w = 0; w < kSortWaves; w++) {
    base += w < wave ? sums[w] : 0;
    total += sums[w];
  }
  __syncthreads();
  *all = total;
  return base + inc - v;
}

struct SortArgs {
  const void* tokens;
  uint32_t* keys;  // tokens of other shards come last, as row n_rows and without a position
  uint32_t* pos;
  uint32_t* used;  // tokens of each row
  uint32_t n, n_rows;
  int64_t first;
  int groups_log2, bins_log2;  // workgroups, rows of one
};

template <typename T>
__global__ __launch_bounds__(kSortThreads) void etha_sort_tokens_kernel(const SortArgs a) {
  constexpr uint32_t kAhead = 8;
  __shared__ uint32_t s_count[kSortWaves << kSortBinsLog2];  // [wave][row]
  __shared__ uint32_t s_noted[kSortWaves][kSortNoted];
  __shared__ uint32_t s_sums[kSortWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), bins = 1u << a.bins_log2;
  const uint32_t group = blockIdx.x, groups = 1u << a.groups_log2;
  const T* tokens = (const T*)a.tokens;
  for (uint32_t i = tid; i < kSortWaves << a.bins_log2; i += kSortThreads) s_count[i] = 0;
  __syncthreads();
  uint32_t* count = s_count + (wave << a.bins_log2);
  uint32_t* noted = s_noted[wave];
  const uint32_t per = (a.n + kSortThreads - 1) / kSortThreads * kWave, lo = wave * per < a.n ? wave * per : a.n;
  const uint32_t hi = a.n - lo < per ? a.n : lo + per;
  // a row, or something from n_rows on; unsigned: an id far below `first` must not wrap into the shard
  const auto row_of = [&](T id) {
    const uint64_t r = (uint64_t)(int64_t)id - (uint64_t)a.first;
    return (int64_t)id >= a.first && r < a.n_rows ? (uint32_t)r : a.n_rows;
  };
  uint32_t lower = 0, n_noted = 0;
  const auto look = [&](T id, bool there, uint32_t p) {
    const uint32_t row = row_of(id), of = row & (groups - 1);
    const bool inside = there && row < a.n_rows, mine = inside && of == group;
    lower += (uint32_t)__popcll(__ballot(inside && of < group));
    const uint64_t mask = __ballot(mine);
    if (!mask) return;
    if (mine) {
      atomicAdd(&count[row >> a.groups_log2], 1u);
      const uint32_t at = n_noted + (uint32_t)__popcll(mask & ((1ull << lane) - 1));
      if (at < kSortNoted) noted[at] = p;
    }
    n_noted += (uint32_t)__popcll(mask);
  };
  uint32_t at = lo;
  for (; at + kAhead * kWave <= hi; at += kAhead * kWave) {
    T id[kAhead];
    #pragma unroll
    for (uint32_t u = 0; u < kAhead; u++) id[u] = tokens[at + u * kWave + lane];
    #pragma unroll
    for (uint32_t u = 0; u < kAhead; u++) look(id[u], true, at + u * kWave + lane);
  }
  for (; at < hi; at += kWave) look(tokens[at + lane < hi ? at + lane : hi - 1], at + lane < hi, at + lane);
  scan_block(lane ? 0 : lower, s_sums, &lower);  // (its barriers stand between the counts and their use, too)
  uint32_t total = 0, inside;
  if (tid < bins)
    for (uint32_t w = 0; w < kSortWaves; w++) total += s_count[(w << a.bins_log2) + tid];
  if (tid < bins && (tid << a.groups_log2 | group) < a.n_rows) a.used[tid << a.groups_log2 | group] = total;
  uint32_t to = lower + scan_block(total, s_sums, &inside);
  if (tid < bins)
    for (uint32_t w = 0; w < kSortWaves; w++) {
      const uint32_t c = s_count[(w << a.bins_log2) + tid];
      s_count[(w << a.bins_log2) + tid] = to;
      to += c;
    }
  __syncthreads();
  // the wave's own tokens in their order: those noted, or all of them once more where there were too many
  volatile uint32_t* place = count;
  const bool all = n_noted > kSortNoted;
  const uint32_t steps = all ? hi - lo : n_noted;
  for (uint32_t i = lane; i < (steps + kWave - 1) / kWave * kWave; i += kWave) {
    const uint32_t p = i < steps ? (all ? lo + i : noted[i]) : a.n;
    const uint32_t row = p < a.n ? row_of(tokens[p]) : a.n_rows, bin = row >> a.groups_log2;
    const bool here = row < a.n_rows && (row & (groups - 1)) == group;
    uint64_t same = __ballot(here);
    if (!same) continue;
    for (int b = 0; b < a.bins_log2; b++) {
      const uint64_t ones = __ballot((bin >> b) & 1);
      same &= (bin >> b) & 1 ? ones : ~ones;
    }
    if (here) {
      const uint32_t before = place[bin], rank = (uint32_t)__popcll(same & ((1ull << lane) - 1));
      __builtin_amdgcn_wave_barrier();
      if ((same >> lane) == 1) place[bin] = before + rank + 1;  // the highest lane of the row
      a.keys[before + rank] = row;
      a.pos[before + rank] = p;
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (group == groups - 1)
    for (uint32_t i = lower + inside + tid; i < a.n; i += kSortThreads) a.keys[i] = a.n_rows;
}

// ---- gradient of the lookup ----------------------------------------------------------------------------------------
// dW[r,:] = scale * sum of the gradient rows whose token is r.  The sorted tokens are cut into chunks of `chunk`
// places; a wave adds up the rows of one chunk for 64 vectors of columns, so that a frequent token is spread over many
// waves.  A row whose tokens all lie in one chunk is written at once; the pieces of a row that crosses chunks go to a
// workspace in fp32 (slot 0 of a chunk: its first row, begun earlier; slot 1: its last row, going on) and are joined in
// chunk order.  Further workgroups of the same launch write the rows that no token names.
struct GradArgs {
  const void* grad;
  void* out;
  const uint32_t* keys;  // sorted
  const uint32_t* pos;
  const uint32_t* used;  // tokens of each row
  float* partial;        // [chunk][2][width]
  uint64_t n, width;
  int64_t grad_stride, out_stride;
  uint32_t n_rows, chunk, n_chunks, n_cols, sum_blocks, zero_blocks;
  uint32_t accumulate;
  float scale;
};

// The columns of a lane.  Vectors that would reach over the end of a row begin earlier, at `at`, so that no load branches:
// their first columns are the neighbour's too and come out the same there.  Rows shorter than a vector (`narrow`) are read
// by elements.
template <int N>
struct Columns {
  uint64_t own, at;
  bool inside, narrow;
  __device__ Columns(uint64_t col, uint64_t width) {
    own = col;
    inside = col < width;
    narrow = width < N;
    at = narrow ? 0 : col + N <= width ? col : width - N;
  }
};

// `count` of K rows of a gradient (the rest repeat the first), all loads on their way at once
template <typename S, int N, int K, typename ROW>
__device__ inline void load_rows(u32x4 (&raw)[K], const GradArgs& a, const Columns<N>& c, uint32_t count, ROW&& row) {
  if (!c.narrow) {
    #pragma unroll
    for (int u = 0; u < K; u++)
      raw[u] = load_raw<16, true>((const typename S::bits*)a.grad + (int64_t)row((uint32_t)u < count ? u : 0) * a.grad_stride + c.at);
  } else {
    #pragma unroll
    for (int u = 0; u < K; u++)
      raw[u] = load_part<sizeof(typename S::bits)>(
          (const char*)((const typename S::bits*)a.grad + (int64_t)row((uint32_t)u < count ? u : 0) * a.grad_stride),
          (int64_t)a.width * (int64_t)sizeof(typename S::bits));
  }
}

// Stored through the caches, unlike the rows of zeros: a wave here writes 1 KB of one row, its neighbours the rest at other
// times, and the lines are put together in L2 (65536 tokens of 4096 into 128256 rows 321 us, 343 us around the caches; 4 tokens
// into 20480 x 2809 fp32 34 us, 70 us).  (These and the following figures: calls with one set of inputs, over and over; the
// first of them takes 334 us where the inputs change from call to call.)
template <typename D, int N>
__device__ inline void write_row(const GradArgs& a, uint32_t row, const Columns<N>& c, float (&acc)[N]) {
  if (!c.inside) return;
  typename D::bits* p = (typename D::bits*)a.out + (int64_t)row * a.out_stride + c.at;
  float v[N];
  if (c.own == c.at && !c.narrow) {
    if (a.accumulate) load_f32<D, N>(v, p, N);
    #pragma unroll
    for (int i = 0; i < N; i++) v[i] = a.accumulate ? v[i] + acc[i] * a.scale : acc[i] * a.scale;
    store_f32<D, N>(p, v, N);
  } else {  // the columns that are this lane's alone
    #pragma unroll
    for (int i = 0; i < N; i++)
      if (c.at + i >= c.own && c.at + i < a.width) p[i] = D::from_f32(a.accumulate ? D::to_f32(p[i]) + acc[i] * a.scale : acc[i] * a.scale);
  }
}

// a piece of a row that crosses chunks, in the workspace
template <int N>
__device__ inline void store_piece(float* piece, const GradArgs& a, const Columns<N>& c, const float (&acc)[N]) {
  if (c.inside) store_f32<F32, N>((uint32_t*)piece + c.at, acc, c.narrow ? (int64_t)a.width : N);
}

// Rows whose loads are on their way at once: 16 in the sums of sorted tokens (20928 x 768: 50 us, 55 us with 8), 8 for few
// tokens, of which most rows have one (509 of 1001 columns: 10.6 us, 12.2 us with 16) and in the join.
constexpr int kGradWaves = 4, kSumAhead = 16, kFewAhead = 8, kJoinAhead = 8;
// Rows that a workgroup looks through for ones without tokens: one a wave, so that they are written in address order by
// workgroups that live as shortly as a copy's (65536 tokens into 128256 x 4096 in bf16: 311 us with 4 rows, 326 us with 64;
// 20928 into 52352 x 768 fp32: 50 us, 62 us).
constexpr uint32_t kZeroRows = 4;

template <typename S>
constexpr int grad_vec() { return 16 / (int)sizeof(typename S::bits); }

template <typename S, typename D>
__global__ __launch_bounds__(kGradWaves* kWave) void etha_embedding_grad_kernel(const GradArgs a) {
  constexpr int N = grad_vec<S>();
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= a.sum_blocks) {  // rows without a token
    for (uint64_t row0 = (uint64_t)(blockIdx.x - a.sum_blocks) * kZeroRows; row0 < a.n_rows; row0 += (uint64_t)a.zero_blocks * kZeroRows) {
      const bool empty = lane < kZeroRows && row0 + lane < a.n_rows && !a.used[row0 + lane];
      uint64_t todo = __ballot(empty);
      constexpr int M = 16 / (int)sizeof(typename D::bits);
      const float zero[M] = {};
      for (uint32_t r = wave; r < kZeroRows; r += kGradWaves)
        if ((todo >> r) & 1) {
          typename D::bits* p = (typename D::bits*)a.out + (int64_t)(row0 + r) * a.out_stride;
          for (uint64_t c = lane * M; c < a.width; c += 64 * M) store_f32<D, M, true>(p + c, zero, (int64_t)(a.width - c));
        }
    }
    return;
  }
  const uint64_t unit = (uint64_t)blockIdx.x * kGradWaves + wave;
  const uint32_t j = (uint32_t)(unit / a.n_cols);
  if (j >= a.n_chunks) return;
  const Columns<N> c((unit % a.n_cols * 64 + lane) * N, a.width);
  const uint64_t begin = (uint64_t)j * a.chunk, end = begin + a.chunk < a.n ? begin + a.chunk : a.n;
  uint32_t cur = a.keys[begin];
  if (cur >= a.n_rows) return;  // other shards' tokens sort behind all rows
  bool open_left = begin && a.keys[begin - 1] == cur;
  float acc[N] = {};
  float* piece = a.partial + (uint64_t)j * 2 * a.width;
  for (uint64_t at = begin; at < end; at += 64) {
    const uint32_t key = at + lane < end ? a.keys[at + lane] : a.n_rows;
    const uint32_t pos = at + lane < end ? a.pos[at + lane] : 0;
    const uint32_t n = (uint32_t)__popcll(__ballot(key < a.n_rows));
    for (uint32_t i = 0; i < n; i += kSumAhead) {
      u32x4 raw[kSumAhead];
      load_rows<S, N>(raw, a, c, n - i, [&](uint32_t u) { return (uint32_t)__builtin_amdgcn_readlane(pos, i + u); });
      #pragma unroll
      for (uint32_t u = 0; u < kSumAhead; u++) {
        if (i + u >= n) break;
        const uint32_t k = __builtin_amdgcn_readlane(key, i + u);
        if (k != cur) {
          if (open_left) store_piece(piece, a, c, acc);
          else write_row<D, N>(a, cur, c, acc);
          open_left = false;
          cur = k;
          #pragma unroll
          for (int e = 0; e < N; e++) acc[e] = 0.f;
        }
        float v[N];
        raw_to_f32<S>(v, raw[u]);
        #pragma unroll
        for (int e = 0; e < N; e++) acc[e] += v[e];
      }
    }
    if (n < 64) break;
  }
  if (open_left) store_piece(piece, a, c, acc);
  else if (end < a.n && a.keys[end] == cur) store_piece(piece + a.width, a, c, acc);
  else write_row<D, N>(a, cur, c, acc);
}

// Few tokens: no sort and one launch.  A workgroup owns 16 rows (and further ones where there are more than a grid takes) and
// 64 vectors of columns; each wave picks the places of its 4 rows' tokens out of all tokens, in their order, and adds their
// rows up.
constexpr uint32_t kFewTokens = 512, kFewTokenRows = 4;

struct FewGradArgs {
  GradArgs g;
  const void* tokens;
  int64_t first;
  uint32_t wide;
};

template <typename S, typename D>
__global__ __launch_bounds__(kGradWaves* kWave) void etha_embedding_grad_few_kernel(const FewGradArgs few) {
  constexpr int N = grad_vec<S>();
  constexpr uint32_t kSteps = kFewTokens / 64;
  const GradArgs& a = few.g;
  __shared__ uint16_t s_list[kGradWaves][kFewTokenRows][kFewTokens];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Columns<N> c(((uint64_t)blockIdx.y * 64 + lane) * N, a.width);
  uint32_t row[kSteps];
  #pragma unroll
  for (uint32_t i = 0; i < kSteps; i++) row[i] = i * 64 + lane < a.n ? local_row(few.tokens, few.wide, i * 64 + lane, few.first, a.n_rows) : a.n_rows;
  for (uint32_t row0 = (blockIdx.x * kGradWaves + wave) * kFewTokenRows; row0 < a.n_rows; row0 += gridDim.x * (kGradWaves * kFewTokenRows)) {
    uint32_t count[kFewTokenRows] = {};
    #pragma unroll
    for (uint32_t i = 0; i < kSteps; i++) {
      if (i * 64 >= a.n) break;
      #pragma unroll
      for (uint32_t r = 0; r < kFewTokenRows; r++) {
        const bool mine = row[i] == row0 + r && row[i] < a.n_rows;
        const uint64_t mask = __ballot(mine);
        if (mine) s_list[wave][r][count[r] + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)(i * 64 + lane);
        count[r] += (uint32_t)__popcll(mask);
      }
    }
    #pragma unroll
    for (uint32_t r = 0; r < kFewTokenRows; r++) {
      if (row0 + r >= a.n_rows || (a.accumulate && !count[r])) continue;
      float acc[N] = {};
      for (uint32_t i = 0; i < count[r]; i += kFewAhead) {
        u32x4 raw[kFewAhead];
        load_rows<S, N>(raw, a, c, count[r] - i, [&](uint32_t u) { return (uint32_t)s_list[wave][r][i + u]; });
        #pragma unroll
        for (uint32_t u = 0; u < kFewAhead; u++) {
          if (i + u >= count[r]) break;
          float v[N];
          raw_to_f32<S>(v, raw[u]);
          #pragma unroll
          for (int e = 0; e < N; e++) acc[e] += v[e];
        }
      }
      write_row<D, N>(a, row0 + r, c, acc);
    }
  }
}

// Rows that cross chunks: the wave of the chunk where such a row begins adds the pieces up.
template <typename S, typename D>
__global__ __launch_bounds__(kGradWaves* kWave) void etha_embedding_join_kernel(const GradArgs a) {
  constexpr int N = grad_vec<S>();
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t unit = (uint64_t)blockIdx.x * kGradWaves + wave;
  uint32_t j = (uint32_t)(unit / a.n_cols);
  if (j >= a.n_chunks) return;
  const Columns<N> c((unit % a.n_cols * 64 + lane) * N, a.width);
  const uint64_t begin = (uint64_t)j * a.chunk, end = begin + a.chunk;
  if (end >= a.n) return;
  const uint32_t key = a.keys[end], last = a.keys[end - 1], first = a.keys[begin], before = begin ? a.keys[begin - 1] : a.n_rows;
  if (key >= a.n_rows || last != key) return;    // nothing goes on behind this chunk
  if (first == key && before == key) return;     // begun earlier
  const int64_t left = c.narrow ? (int64_t)a.width : N;
  float acc[N];
  load_f32<F32, N>(acc, (const uint32_t*)(a.partial + ((uint64_t)j * 2 + 1) * a.width + c.at), left);
  // the chunks behind this one that begin with the same row, 64 at a time
  for (;;) {
    const uint64_t start = (uint64_t)(j + 1 + lane) * a.chunk;
    const uint64_t same = __ballot(start < a.n && a.keys[start < a.n ? start : 0] == key);
    const uint32_t more = ~same ? __builtin_ctzll(~same) : 64;
    for (uint32_t i = 0; i < more; i += kJoinAhead) {
      u32x4 raw[kJoinAhead][N / 4];
      if (!c.narrow) {
        #pragma unroll
        for (uint32_t u = 0; u < kJoinAhead; u++)
          #pragma unroll
          for (int e = 0; e < N / 4; e++)
            raw[u][e] = load_raw<16>(a.partial + (uint64_t)(j + 1 + (i + u < more ? i + u : i)) * 2 * a.width + c.at + e * 4);
      } else {
        #pragma unroll
        for (uint32_t u = 0; u < kJoinAhead; u++)
          #pragma unroll
          for (int e = 0; e < N / 4; e++)
            raw[u][e] = load_part<4>((const char*)(a.partial + (uint64_t)(j + 1 + (i + u < more ? i + u : i)) * 2 * a.width + e * 4),
                                     ((int64_t)a.width - e * 4) * 4);
      }
      #pragma unroll
      for (uint32_t u = 0; u < kJoinAhead; u++) {
        if (i + u >= more) break;
        #pragma unroll
        for (int e = 0; e < N; e++) acc[e] += __builtin_bit_cast(float, (uint32_t)raw[u][e / 4][e % 4]);
      }
    }
    j += more;
    if (more < 64) break;
  }
  write_row<D, N>(a, key, c, acc);
}

// ---- rows to 8 bits --------------------------------------------------------------------------------------------
// The row stays in registers between its maximum and its conversion (RowScale), so it is read once.
struct QuantArgs {
  const void* x;
  int8_t* values;
  float* scales;
  uint64_t rows, width;
  int64_t x_stride, values_stride;
};

// THREADS work-items a row.  The last 8 elements of a row whose width is no multiple of 8 overlap those before, so that no
// load branches: both come out the same.  (Rows shorter than 8 go by elements.)
template <typename S, int THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS) void etha_quantize_rows_kernel(const QuantArgs a) {
  constexpr int kBlock = THREADS < 256 ? 256 : THREADS, kWaves = THREADS / kWave, kPieces = 8 * (int)sizeof(typename S::bits) / 16;
  constexpr int kPer = 8 / kPieces;
  __shared__ uint32_t s_max[kBlock / kWave];
  const uint32_t tid = threadIdx.x % THREADS;
  const uint64_t row = (uint64_t)blockIdx.x * (kBlock / THREADS) + threadIdx.x / THREADS;
  const bool there = row < a.rows;
  const typename S::bits* x = (const typename S::bits*)a.x + (int64_t)(there ? row : a.rows - 1) * a.x_stride;
  int8_t* out = a.values + (int64_t)row * a.values_stride;
  const int64_t width = (int64_t)a.width, last = width - 8, span = (int64_t)THREADS * CHUNKS * 8;
  u32x4 raw[CHUNKS][kPieces];
  const auto load = [&](int64_t base) {
    if (width >= 8) {
      #pragma unroll
      for (int c = 0; c < CHUNKS; c++) {
        const int64_t at = base + ((int64_t)c * THREADS + tid) * 8;
        #pragma unroll
        for (int i = 0; i < kPieces; i++) raw[c][i] = load_raw<16, true>(x + (at < last ? at : last) + i * kPer);
      }
    } else {
      #pragma unroll
      for (int c = 0; c < CHUNKS; c++)
        #pragma unroll
        for (int i = 0; i < kPieces; i++)
          raw[c][i] = load_part<sizeof(typename S::bits)>((const char*)(x + i * kPer), (width - i * kPer) * (int64_t)sizeof(typename S::bits));
    }
  };
  const auto values = [&](int c, float (&v)[8]) {
    #pragma unroll
    for (int i = 0; i < kPieces; i++) {
      float part[kPer];
      raw_to_f32<S>(part, raw[c][i]);
      #pragma unroll
      for (int e = 0; e < kPer; e++) v[i * kPer + e] = part[e];
    }
  };
  uint32_t top = 0;
  for (int64_t base = 0; base < width; base += span) {
    load(base);
    #pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
      float v[8];
      values(c, v);
      top = largest_bits(v, top);
    }
  }
  top = group_max<THREADS < kWave ? THREADS : kWave>(top);
  if constexpr (kWaves > 1) {
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = top;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < kWaves; w++) top = s_max[w] > top ? s_max[w] : top;
  }
  if (!there) return;
  const RowScale scale(top);
  for (int64_t base = 0; base < width; base += span) {
    if (width > span) load(base);
    #pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
      const int64_t at = base + ((int64_t)c * THREADS + tid) * 8;
      if (at >= width) continue;
      float v[8];
      values(c, v);
      const u32x2 packed = scale.pack<S>(v);
      if (width >= 8) {
        store_raw<8, true>(out + (at < last ? at : last), packed);
      } else {
        for (int i = 0; i < 8; i++)
          if (i < width) out[i] = (int8_t)(packed[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
  if (tid == 0) a.scales[row] = scale.scale;
}

// ---- host side ---------------------------------------------------------------------------------------------------
int es_of(uint32_t dtype) { return dtype == ETHA_F32 ? 4 : dtype == ETHA_BF16 || dtype == ETHA_F16 ? 2 : 0; }

int log2_up(uint64_t x) {
  int l = 0;
  while (l < 63 && (1ull << l) < x) l++;
  return l;
}

int check_tokens(const char* what, const void* tokens, uint32_t token_dtype, uint64_t n_tokens, uint64_t n_rows, uint64_t width) {
  if (token_dtype != ETHA_I32 && token_dtype != ETHA_I64) return fail(ETHA_ERR_INVALID, "%s: tokens are 32- or 64-bit integers", what);
  if (n_tokens && !tokens) return fail(ETHA_ERR_INVALID, "%s: null tokens", what);
  if (n_tokens >= 1ull << 31) return fail(ETHA_ERR_UNSUPPORTED, "%s: %llu tokens; at most 2^31 - 1", what, (unsigned long long)n_tokens);
  if (n_rows >= 1ull << 31) return fail(ETHA_ERR_UNSUPPORTED, "%s: %llu rows; at most 2^31 - 1", what, (unsigned long long)n_rows);
  if (width > 1ull << 24) return fail(ETHA_ERR_UNSUPPORTED, "%s: width %llu; at most 2^24", what, (unsigned long long)width);
  return ETHA_OK;
}

// Workgroups of the sort: one a CU, more where a workgroup's rows would need more LDS than there is.
int sort_groups_log2(uint64_t n_rows) {
  const int rows = log2_up(n_rows);
  return rows < kSortGroupsLog2 ? rows : rows - kSortGroupsLog2 > kSortBinsLog2 ? rows - kSortBinsLog2 : kSortGroupsLog2;
}
// Each of them looks through all tokens: 2^36 looks are some 50 ms.
int check_gradient_tokens(const char* what, uint64_t n_tokens, uint64_t n_rows) {
  if (n_tokens > 1ull << 26 || (n_tokens > kFewTokens && n_tokens << sort_groups_log2(n_rows) > 1ull << 36))
    return fail(ETHA_ERR_UNSUPPORTED, "%s: %llu tokens of %llu rows; at most 2^26 tokens, or 2^46 over the rows where those are more than 2^20",
                what, (unsigned long long)n_tokens, (unsigned long long)n_rows);
  return ETHA_OK;
}

// Workgroups that sum, and that write rows of zeros: with 256 work-items each, together in a grid of fewer than 2^32.
constexpr uint32_t kMostGradBlocks = 1u << 23;

// Column blocks, chunk length and workspace of a gradient call: a rule on sizes alone.
struct GradPlan {
  uint32_t n_cols, chunk, n_chunks;
  int groups_log2, bins_log2;
  uint64_t keys_bytes, used_bytes, partial_bytes;
  uint64_t total() const { return 2 * keys_bytes + used_bytes + partial_bytes; }
};
GradPlan grad_plan(uint64_t n, uint64_t n_rows, uint64_t width, int es) {
  GradPlan p = {};
  const uint64_t per = 64 * (16 / es);
  p.n_cols = (uint32_t)((width + per - 1) / per);
  // chunks of 128 places, shorter while there would be fewer waves than the chip holds a few of per SIMD (16 places where that
  // is still less than two waves a SIMD: 6965 tokens of 76 columns 23 us, 28 us with 32; 57984 of 128 columns 56 us, 48 us with
  // 32); such chunks make fewer than 8192 waves, so their pieces need at most 32 MB of workspace.  Chunks of 128 get longer where
  // there would be more than 2048 of them.  What the call takes does not jump there, though the number of waves does: 524160
  // tokens of 512 columns (8190 chunks of 64) 807 us, 524544 (2050 chunks of 256) 780 us; 262016 of 1024 columns 427 us, 262400
  // 410 us.
  uint64_t chunk = 128;
  while (chunk > 32 && (n + chunk - 1) / chunk * p.n_cols < 4096) chunk >>= 1;
  if (chunk == 32 && (n + 15) / 16 * p.n_cols < 2048) chunk = 16;
  if ((n + chunk - 1) / chunk > 2048 && chunk == 128) chunk = ((n + 2047) / 2048 + 127) / 128 * 128;
  p.chunk = (uint32_t)chunk;
  p.n_chunks = (uint32_t)((n + chunk - 1) / chunk);
  p.groups_log2 = sort_groups_log2(n_rows);
  p.bins_log2 = log2_up(n_rows) - p.groups_log2;
  const auto up = [](uint64_t b) { return (b + 255) / 256 * 256; };
  p.keys_bytes = up(n * 4);
  p.used_bytes = up(n_rows * 4);
  p.partial_bytes = up((uint64_t)p.n_chunks * 2 * width * 4);
  return p;
}

template <typename S, int THREADS, int CHUNKS>
void quantize_with(const QuantArgs& a, hipStream_t stream) {
  constexpr int kBlock = THREADS < 256 ? 256 : THREADS, kRows = kBlock / THREADS;
  hipLaunchKernelGGL((etha_quantize_rows_kernel<S, THREADS, CHUNKS>), dim3((uint32_t)((a.rows + kRows - 1) / kRows)), dim3(kBlock), 0, stream, a);
}

// Part of a wave or a wave a row while the row fits its registers (narrow rows: 45913 of 102 in bf16 6 us, 36 us with a wave),
// else a workgroup a row, always with little more room than the row needs (64128 rows of 4096 in fp32: 215 us with room for
// 4096, some 15 us more with room for 8192).  16-bit rows go further in a wave: 49268 of 832 31 us with 32 lanes, 33 us with 64;
// 23040 of 2496 36 us with a wave, 48 us with a workgroup; 32768 of 2700 59 us, 71 us.  From 3585 to 4096 that depends on the
// rows.  bf16, 3600 wide, a wave and a workgroup: 8192 rows 27.7 and 23.5 us, 16384 43.2 and 41.3, 24576 59.1 and 59.4, 32768
// 75.2 and 77.7, 64128 137 and 148 us; fp16: 24576 rows 56.3 and 53.7 us, 32768 71.0 and 69.8, 49152 101.5 and 102.4, 64128 130.3
// and 131.8 us; 4096 wide alike.  One cut for both types, at 32768 rows, is within 6 % of the better one wherever it was measured
// (farthest: fp16, 32768 of 3848, 75.5 and 71.6 us).  fp32 does not go further in a wave: 49268 of 832 38 us with 32 lanes, 36 us;
// 8246 of 2453 22.3 us with a wave, 20.7 us.
int quantize_launch(const QuantArgs& a, uint32_t dtype, hipStream_t stream) {
  with_type(dtype, [&](auto s) {
    typedef decltype(s) S;
    if constexpr (sizeof(typename S::bits) == 2) {
      if (a.width > 16 * 8 * 4 && a.width <= 32 * 8 * 4) return quantize_with<S, 32, 4>(a, stream);
      if (a.width > 64 * 8 * 4 && a.width <= 64 * 8 * 5) return quantize_with<S, 64, 5>(a, stream);
      if (a.width > 64 * 8 * 5 && a.width <= 64 * 8 * 8 && (a.width <= 64 * 8 * 7 || a.rows >= 32768)) return quantize_with<S, 64, 8>(a, stream);
    } else {
      if (a.width > 16 * 8 * 4 && a.width <= 64 * 8 * 2) return quantize_with<S, 64, 2>(a, stream);
    }
    if (a.width <= 16 * 8 * 4) return quantize_with<S, 16, 4>(a, stream);
    if (a.width <= 64 * 8 * 4) return quantize_with<S, 64, 4>(a, stream);
    if (a.width <= 256 * 8 * 2) return quantize_with<S, 256, 2>(a, stream);
    if (a.width <= 256 * 8 * 4) return quantize_with<S, 256, 4>(a, stream);
    return quantize_with<S, 1024, 4>(a, stream);
  });
  return launched("etha_quantize_rows_kernel");
}

}  // namespace

extern "C" {

int etha_embedding(const void* tokens, uint32_t token_dtype, uint64_t n_tokens, const void* weight, uint32_t weight_dtype,
                   uint64_t n_rows, uint64_t width, int64_t weight_stride, int64_t first_row, float scale, void* out,
                   uint32_t out_dtype, int64_t out_stride, void* stream) {
  const int rc = check_tokens("etha_embedding", tokens, token_dtype, n_tokens, n_rows, width);
  if (rc != ETHA_OK) return rc;
  const int es = es_of(weight_dtype), eo = es_of(out_dtype);
  if (!es || !eo) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding: element types are f32, bf16 and f16");
  if (!n_tokens || !width) return ETHA_OK;
  if ((!weight && n_rows) || !out) return fail(ETHA_ERR_INVALID, "etha_embedding: null tensor");
  LookupArgs a = {tokens, weight, out, n_tokens, width, first_row, weight_stride, out_stride, (uint32_t)n_rows, 0,
                  token_dtype == ETHA_I64, scale};
  const uint64_t n = lookup_vec(es, eo), vecs = (width + n - 1) / n;
  a.lanes_log2 = (uint32_t)log2_up(vecs < 256 ? vecs : 256);
  const uint32_t per_block = 256u >> a.lanes_log2;
  uint64_t gx = (n_tokens + per_block - 1) / per_block;
  if (gx > 1u << 22) gx = 1u << 22;
  const dim3 grid((uint32_t)gx, (uint32_t)((vecs + (1u << a.lanes_log2) - 1) >> a.lanes_log2));
  if (grid.y > 65535) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding: width %llu is too large", (unsigned long long)width);
  with_type(weight_dtype, [&](auto s) {
    with_type(out_dtype, [&](auto d) {
      hipLaunchKernelGGL((etha_embedding_kernel<decltype(s), decltype(d)>), grid, dim3(256), 0, (hipStream_t)stream, a);
    });
  });
  return launched("etha_embedding_kernel");
}

int etha_embedding_grad_workspace(uint64_t n_tokens, uint64_t n_rows, uint64_t width, uint32_t grad_dtype, uint64_t* bytes) {
  int rc = check_tokens("etha_embedding_grad_workspace", &n_tokens, ETHA_I32, n_tokens, n_rows, width);
  if (rc == ETHA_OK) rc = check_gradient_tokens("etha_embedding_grad_workspace", n_tokens, n_rows);
  if (rc != ETHA_OK) return rc;
  if (!bytes) return fail(ETHA_ERR_INVALID, "etha_embedding_grad_workspace: null result");
  if (!es_of(grad_dtype)) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad_workspace: element types are f32, bf16 and f16");
  *bytes = n_tokens > kFewTokens && n_rows && width ? grad_plan(n_tokens, n_rows, width, es_of(grad_dtype)).total() : 0;
  return ETHA_OK;
}

int etha_embedding_grad(const void* grad, uint32_t grad_dtype, int64_t grad_stride, const void* tokens, uint32_t token_dtype,
                        uint64_t n_tokens, uint64_t n_rows, uint64_t width, int64_t first_row, float scale, void* out,
                        uint32_t out_dtype, int64_t out_stride, int accumulate, void* workspace, uint64_t workspace_bytes,
                        void* stream) {
  int rc = check_tokens("etha_embedding_grad", tokens, token_dtype, n_tokens, n_rows, width);
  if (rc == ETHA_OK) rc = check_gradient_tokens("etha_embedding_grad", n_tokens, n_rows);
  if (rc != ETHA_OK) return rc;
  const int es = es_of(grad_dtype);
  if (!es || !es_of(out_dtype)) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: element types are f32, bf16 and f16");
  if (!n_rows || !width || (!n_tokens && accumulate)) return ETHA_OK;
  if (!out || (n_tokens && !grad)) return fail(ETHA_ERR_INVALID, "etha_embedding_grad: null tensor");
  GradArgs g = {};
  g.out = out;
  g.grad = grad;
  g.n = n_tokens;
  g.width = width;
  g.grad_stride = grad_stride;
  g.out_stride = out_stride;
  g.n_rows = (uint32_t)n_rows;
  g.accumulate = accumulate != 0;
  g.scale = scale;
  g.chunk = g.n_cols = 1;
  if (n_tokens <= kFewTokens) {
    const FewGradArgs few = {g, tokens, first_row, token_dtype == ETHA_I64};
    const uint64_t per = 64 * (16 / es);
    dim3 grid((uint32_t)((n_rows + kGradWaves * kFewTokenRows - 1) / (kGradWaves * kFewTokenRows)), (uint32_t)((width + per - 1) / per));
    if (grid.y > 65535) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: too many columns");
    if (grid.x > kMostGradBlocks) grid.x = kMostGradBlocks;  // which then go round
    with_type(grad_dtype, [&](auto s) {
      with_type(out_dtype, [&](auto d) {
        hipLaunchKernelGGL((etha_embedding_grad_few_kernel<decltype(s), decltype(d)>), grid, dim3(kGradWaves * kWave), 0,
                           (hipStream_t)stream, few);
      });
    });
    return launched("etha_embedding_grad_few_kernel");
  }
  {
    const GradPlan p = grad_plan(n_tokens, n_rows, width, es);
    if (!workspace || workspace_bytes < p.total() || ((uintptr_t)workspace & 15))
      return fail(ETHA_ERR_INVALID, "etha_embedding_grad: the workspace has to hold %llu bytes at a 16-byte address",
                  (unsigned long long)p.total());
    SortArgs sort = {tokens, (uint32_t*)workspace, nullptr, nullptr, (uint32_t)n_tokens, (uint32_t)n_rows, first_row, p.groups_log2, p.bins_log2};
    sort.pos = (uint32_t*)((char*)sort.keys + p.keys_bytes);
    sort.used = (uint32_t*)((char*)sort.pos + p.keys_bytes);
    const auto kernel = token_dtype == ETHA_I64 ? etha_sort_tokens_kernel<int64_t> : etha_sort_tokens_kernel<int32_t>;
    hipLaunchKernelGGL(kernel, dim3(1u << p.groups_log2), dim3(kSortThreads), 0, (hipStream_t)stream, sort);
    if ((rc = launched("etha_sort_tokens_kernel")) != ETHA_OK) return rc;
    g.keys = sort.keys;
    g.pos = sort.pos;
    g.used = sort.used;
    g.partial = (float*)((char*)sort.used + p.used_bytes);
    g.chunk = p.chunk;
    g.n_chunks = p.n_chunks;
    g.n_cols = p.n_cols;
    const uint64_t blocks = ((uint64_t)p.n_chunks * p.n_cols + kGradWaves - 1) / kGradWaves;
    if (blocks > kMostGradBlocks) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: too many tokens for this width");
    g.sum_blocks = (uint32_t)blocks;
  }
  const uint64_t zero_blocks = accumulate ? 0 : (n_rows + kZeroRows - 1) / kZeroRows;
  g.zero_blocks = (uint32_t)(zero_blocks < kMostGradBlocks ? zero_blocks : kMostGradBlocks - 1);  // which then go round
  with_type(grad_dtype, [&](auto s) {
    with_type(out_dtype, [&](auto d) {
      hipLaunchKernelGGL((etha_embedding_grad_kernel<decltype(s), decltype(d)>), dim3(g.sum_blocks + g.zero_blocks),
                         dim3(kGradWaves * kWave), 0, (hipStream_t)stream, g);
    });
  });
  if ((rc = launched("etha_embedding_grad_kernel")) != ETHA_OK) return rc;
  if (g.n_chunks < 2) return ETHA_OK;  // nothing can cross
  with_type(grad_dtype, [&](auto s) {
    with_type(out_dtype, [&](auto d) {
      hipLaunchKernelGGL((etha_embedding_join_kernel<decltype(s), decltype(d)>), dim3(g.sum_blocks), dim3(kGradWaves * kWave), 0,
                         (hipStream_t)stream, g);
    });
  });
  return launched("etha_embedding_join_kernel");
}

int etha_quantize_rows(const void* x, uint32_t dtype, uint64_t rows, uint64_t width, int64_t x_stride, int8_t* values,
                       int64_t values_stride, float* scales, void* stream) {
  if (!es_of(dtype)) return fail(ETHA_ERR_UNSUPPORTED, "etha_quantize_rows: element types are f32, bf16 and f16");
  if (!rows) return ETHA_OK;
  if ((width && (!x || !values)) || !scales) return fail(ETHA_ERR_INVALID, "etha_quantize_rows: null tensor");
  if (rows >= 1ull << 31) return fail(ETHA_ERR_UNSUPPORTED, "etha_quantize_rows: %llu rows; at most 2^31 - 1", (unsigned long long)rows);
  constexpr uint64_t kMostRows = 1u << 21;  // of a launch: a grid has fewer than 2^32 work-items, up to 1024 of them a row
  for (uint64_t done = 0; done < rows; done += kMostRows) {
    const int rc = quantize_launch({(const char*)x + (int64_t)done * x_stride * es_of(dtype), values + (int64_t)done * values_stride,
                                    scales + done, rows - done < kMostRows ? rows - done : kMostRows, width, x_stride, values_stride},
                                   dtype, (hipStream_t)stream);
    if (rc != ETHA_OK) return rc;
  }
  return ETHA_OK;
}

}  // extern "C"
