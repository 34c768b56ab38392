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
// A stable radix sort of (row, position), digits of up to 9 bits, so that a row's positions come in their own order
// and the sums that follow do not depend on timing.  A wave ranks 64 keys at a time: the lanes with the same digit
// find each other with one ballot per digit bit, and the wave's running count of the digit lies in LDS.
constexpr int kMaxBins = 512;
constexpr uint32_t kOneBlockThreads = 1024, kOneBlockTokens = 8192;
constexpr uint32_t kSortThreads = 256;
// Tokens of a workgroup where there are more: every workgroup adds up the counts of all of them, so they get longer where
// there would be more than 256 (65536 tokens: a pass takes 11 us with 64 workgroups, 29 us with 16).
constexpr uint32_t sort_tokens(uint64_t n) { return n <= 256 * 1024 ? 1024 : 4096; }

__device__ inline uint64_t same_digit(uint32_t digit, int bits) {
  uint64_t mask = ~0ull;
  for (int b = 0; b < bits; b++) {
    const uint64_t ones = __ballot((digit >> b) & 1);
    mask &= (digit >> b) & 1 ? ones : ~ones;
  }
  return mask;
}

// Rank of this lane's key among the wave's earlier keys of the same digit; `counts` (the wave's own, in LDS) goes on.
__device__ inline uint32_t rank_in_wave(volatile uint16_t* counts, uint32_t digit, int bits) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t mask = same_digit(digit, bits);
  const uint32_t before = counts[digit];
  __builtin_amdgcn_wave_barrier();
  if ((mask >> lane) == 1) counts[digit] = (uint16_t)(before + __popcll(mask));  // the highest lane of the digit
  __builtin_amdgcn_wave_barrier();
  return before + __popcll(mask & ((1ull << lane) - 1));
}

// Exclusive sum over the workgroup's work-items; `sums` holds one word per wave.
__device__ inline uint32_t scan_block(uint32_t v, uint32_t* sums) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = v;
  #pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(inc, d);
    if (lane >= (uint32_t)d) inc += o;
  }
  if (lane == 63) sums[wave] = inc;
  __syncthreads();
  uint32_t base = 0;
  for (uint32_t w = 0; w < wave; w++) base += sums[w];
  __syncthreads();
  return base + inc - v;
}

// Up to kOneBlockTokens tokens: all passes in one workgroup.
__global__ __launch_bounds__(kOneBlockThreads) void etha_sort_tokens_kernel(const void* tokens, uint32_t wide, uint32_t n, int64_t first,
                                                                          uint32_t n_rows, int passes, int bits, uint32_t* keys_out,
                                                                          uint32_t* pos_out) {
  constexpr uint32_t kWaves = kOneBlockThreads / kWave, kItems = kOneBlockTokens / kOneBlockThreads;
  __shared__ uint32_t s_key[kOneBlockTokens];
  __shared__ uint16_t s_pos[kOneBlockTokens];
  __shared__ uint16_t s_count[kWaves][kMaxBins];
  __shared__ uint32_t s_base[kMaxBins];
  __shared__ uint32_t s_sums[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t items = (n + kOneBlockThreads - 1) / kOneBlockThreads;  // per work-item, at most kItems
  const uint32_t at0 = wave * items * 64 + lane;
  uint32_t key[kItems], pos[kItems];
  #pragma unroll
  for (uint32_t i = 0; i < kItems; i++) {
    const uint32_t p = at0 + i * 64;
    pos[i] = p;
    key[i] = 0xffffffffu;  // behind the last token: sorts behind everything
    if (i < items && p < n) key[i] = local_row(tokens, wide, p, first, n_rows);
  }
  const uint32_t bins = 1u << bits;
  for (int pass = 0; pass < passes; pass++) {
    const int shift = pass * bits;
    for (uint32_t i = tid; i < kWaves * kMaxBins; i += kOneBlockThreads) (&s_count[0][0])[i] = 0;
    __syncthreads();
    uint32_t rank[kItems];
    #pragma unroll
    for (uint32_t i = 0; i < kItems; i++)
      if (i < items) rank[i] = rank_in_wave(s_count[wave], (key[i] >> shift) & (bins - 1), bits);
    __syncthreads();
    uint32_t total = 0;
    if (tid < bins)
      for (uint32_t w = 0; w < kWaves; w++) {
        const uint32_t c = s_count[w][tid];
        s_count[w][tid] = (uint16_t)total;
        total += c;
      }
    const uint32_t base = scan_block(total, s_sums);
    if (tid < bins) s_base[tid] = base;
    __syncthreads();
    #pragma unroll
    for (uint32_t i = 0; i < kItems; i++)
      if (i < items) {
        const uint32_t digit = (key[i] >> shift) & (bins - 1);
        const uint32_t to = s_base[digit] + s_count[wave][digit] + rank[i];
        s_key[to] = key[i];
        s_pos[to] = (uint16_t)pos[i];
      }
    __syncthreads();
    #pragma unroll
    for (uint32_t i = 0; i < kItems; i++)
      if (i < items) {
        key[i] = s_key[at0 + i * 64];
        pos[i] = s_pos[at0 + i * 64];
      }
    __syncthreads();
  }
  #pragma unroll
  for (uint32_t i = 0; i < kItems; i++) {
    const uint32_t p = at0 + i * 64;
    if (i < items && p < n) {
      keys_out[p] = key[i];
      pos_out[p] = pos[i];
    }
  }
}

struct SortArgs {
  const void* tokens;     // first pass: keys come from the tokens, positions are the places themselves
  const uint32_t* keys_in;
  const uint32_t* pos_in;
  uint32_t* keys_out;
  uint32_t* pos_out;
  uint32_t* hist;         // [block][bin]
  uint64_t n;
  int64_t first;
  uint32_t n_rows, wide;
  int shift, bits;
};

__device__ inline uint32_t sort_key(const SortArgs& a, uint64_t p) {
  if (p >= a.n) return 0xffffffffu;
  return a.keys_in ? a.keys_in[p] : local_row(a.tokens, a.wide, p, a.first, a.n_rows);
}

template <uint32_t TOKENS>
__global__ __launch_bounds__(kSortThreads) void etha_sort_count_kernel(const SortArgs a) {
  __shared__ uint32_t s_count[kMaxBins];
  const uint32_t bins = 1u << a.bits;
  for (uint32_t i = threadIdx.x; i < bins; i += kSortThreads) s_count[i] = 0;
  __syncthreads();
  const uint64_t base = (uint64_t)blockIdx.x * TOKENS;
  for (uint32_t i = threadIdx.x; i < TOKENS; i += kSortThreads)
    if (base + i < a.n) atomicAdd(&s_count[(sort_key(a, base + i) >> a.shift) & (bins - 1)], 1u);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < bins; i += kSortThreads) a.hist[(uint64_t)blockIdx.x * bins + i] = s_count[i];
}

template <uint32_t TOKENS>
__global__ __launch_bounds__(kSortThreads) void etha_sort_scatter_kernel(const SortArgs a) {
  constexpr uint32_t kWaves = kSortThreads / kWave, kItems = TOKENS / kSortThreads;
  constexpr uint32_t kBinsPer = kMaxBins / kSortThreads;
  __shared__ uint16_t s_count[kWaves][kMaxBins];
  __shared__ uint32_t s_base[kMaxBins];
  __shared__ uint32_t s_sums[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1u << a.bits;
  for (uint32_t i = tid; i < kWaves * kMaxBins; i += kSortThreads) (&s_count[0][0])[i] = 0;
  // where this block's keys of each bin begin: all keys of lower bins, then the earlier blocks' of this bin
  uint32_t before[kBinsPer], total[kBinsPer], sum = 0;
  #pragma unroll
  for (uint32_t j = 0; j < kBinsPer; j++) {
    const uint32_t bin = tid * kBinsPer + j;
    before[j] = total[j] = 0;
    if (bin < bins) {
      #pragma unroll 8
      for (uint32_t b = 0; b < gridDim.x; b++) {
        const uint32_t c = a.hist[(uint64_t)b * bins + bin];
        before[j] += b < blockIdx.x ? c : 0;
        total[j] += c;
      }
    }
    sum += total[j];
  }
  uint32_t base = scan_block(sum, s_sums);
  #pragma unroll
  for (uint32_t j = 0; j < kBinsPer; j++) {
    const uint32_t bin = tid * kBinsPer + j;
    if (bin < bins) s_base[bin] = base + before[j];
    base += total[j];
  }
  __syncthreads();
  const uint64_t at0 = (uint64_t)blockIdx.x * TOKENS + wave * (kItems * 64) + lane;
  uint32_t key[kItems], rank[kItems];
  #pragma unroll
  for (uint32_t i = 0; i < kItems; i++) key[i] = sort_key(a, at0 + i * 64);
  #pragma unroll
  for (uint32_t i = 0; i < kItems; i++) rank[i] = rank_in_wave(s_count[wave], (key[i] >> a.shift) & (bins - 1), a.bits);
  __syncthreads();
  for (uint32_t bin = tid; bin < bins; bin += kSortThreads) {
    uint32_t sofar = 0;
    for (uint32_t w = 0; w < kWaves; w++) {
      const uint32_t c = s_count[w][bin];
      s_count[w][bin] = (uint16_t)sofar;
      sofar += c;
    }
  }
  __syncthreads();
  #pragma unroll
  for (uint32_t i = 0; i < kItems; i++) {
    const uint64_t p = at0 + i * 64;
    if (p < a.n) {
      const uint32_t digit = (key[i] >> a.shift) & (bins - 1);
      const uint32_t to = s_base[digit] + s_count[wave][digit] + rank[i];
      a.keys_out[to] = key[i];
      a.pos_out[to] = a.pos_in ? a.pos_in[p] : (uint32_t)p;
    }
  }
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
  float* partial;        // [chunk][2][width]
  uint64_t n, width;
  int64_t grad_stride, out_stride;
  uint32_t n_rows, chunk, n_chunks, n_cols, sum_blocks;
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
// into 20480 x 2809 fp32 34 us, 70 us).
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

constexpr int kGradWaves = 4, kGradAhead = 8;
// Rows that a workgroup looks through for ones without tokens: one a wave, so that they are written in address order by
// workgroups that live as shortly as a copy's (128256 x 4096 in bf16: 327 us with 4 rows, 357 us with 64).
constexpr uint32_t kZeroRows = 4;

template <typename S>
constexpr int grad_vec() { return 16 / (int)sizeof(typename S::bits); }

template <typename S, typename D>
__global__ __launch_bounds__(kGradWaves* kWave) void etha_embedding_grad_kernel(const GradArgs a) {
  constexpr int N = grad_vec<S>();
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x >= a.sum_blocks) {  // rows without a token
    const uint64_t row0 = (uint64_t)(blockIdx.x - a.sum_blocks) * kZeroRows;
    uint64_t lo = 0, hi = a.n;
    const uint32_t mine = (uint32_t)(row0 + lane);
    while (lo < hi) {
      const uint64_t mid = (lo + hi) >> 1;
      if (a.keys[mid] < mine) lo = mid + 1; else hi = mid;
    }
    const bool empty = lane < kZeroRows && row0 + lane < a.n_rows && !(lo < a.n && a.keys[lo] == mine);
    uint64_t todo = __ballot(empty);
    constexpr int M = 16 / (int)sizeof(typename D::bits);
    const float zero[M] = {};
    for (uint32_t r = wave; r < kZeroRows; r += kGradWaves)
      if ((todo >> r) & 1) {
        typename D::bits* p = (typename D::bits*)a.out + (int64_t)(row0 + r) * a.out_stride;
        for (uint64_t c = lane * M; c < a.width; c += 64 * M) store_f32<D, M, true>(p + c, zero, (int64_t)(a.width - c));
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
    for (uint32_t i = 0; i < n; i += kGradAhead) {
      u32x4 raw[kGradAhead];
      load_rows<S, N>(raw, a, c, n - i, [&](uint32_t u) { return (uint32_t)__builtin_amdgcn_readlane(pos, i + u); });
      #pragma unroll
      for (uint32_t u = 0; u < kGradAhead; u++) {
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

// Few tokens: no sort and one launch.  A workgroup owns 16 rows and 64 vectors of columns; each wave picks the places of
// its 4 rows' tokens out of all tokens, in their order, and adds their rows up.
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
  const uint32_t row0 = (blockIdx.x * kGradWaves + wave) * kFewTokenRows;
  const Columns<N> c(((uint64_t)blockIdx.y * 64 + lane) * N, a.width);
  uint32_t row[kSteps];
  #pragma unroll
  for (uint32_t i = 0; i < kSteps; i++) row[i] = i * 64 + lane < a.n ? local_row(few.tokens, few.wide, i * 64 + lane, few.first, a.n_rows) : a.n_rows;
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
    for (uint32_t i = 0; i < count[r]; i += kGradAhead) {
      u32x4 raw[kGradAhead];
      load_rows<S, N>(raw, a, c, count[r] - i, [&](uint32_t u) { return (uint32_t)s_list[wave][r][i + u]; });
      #pragma unroll
      for (uint32_t u = 0; u < kGradAhead; u++) {
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
  constexpr int kAhead = N > 4 ? 4 : 8;
  const int64_t left = c.narrow ? (int64_t)a.width : N;
  float acc[N];
  load_f32<F32, N>(acc, (const uint32_t*)(a.partial + ((uint64_t)j * 2 + 1) * a.width + c.at), left);
  // the chunks behind this one that begin with the same row, 64 at a time
  for (;;) {
    const uint64_t start = (uint64_t)(j + 1 + lane) * a.chunk;
    const uint64_t same = __ballot(start < a.n && a.keys[start < a.n ? start : 0] == key);
    const uint32_t more = ~same ? __builtin_ctzll(~same) : 64;
    for (uint32_t i = 0; i < more; i += kAhead) {
      u32x4 raw[kAhead][N / 4];
      if (!c.narrow) {
        #pragma unroll
        for (uint32_t u = 0; u < kAhead; u++)
          #pragma unroll
          for (int e = 0; e < N / 4; e++)
            raw[u][e] = load_raw<16>(a.partial + (uint64_t)(j + 1 + (i + u < more ? i + u : i)) * 2 * a.width + c.at + e * 4);
      } else {
        #pragma unroll
        for (uint32_t u = 0; u < kAhead; u++)
          #pragma unroll
          for (int e = 0; e < N / 4; e++)
            raw[u][e] = load_part<4>((const char*)(a.partial + (uint64_t)(j + 1 + (i + u < more ? i + u : i)) * 2 * a.width + e * 4),
                                     ((int64_t)a.width - e * 4) * 4);
      }
      #pragma unroll
      for (uint32_t u = 0; u < kAhead; u++) {
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
      const u32x2 packed = scale.pack(v);
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

// Of a gradient, whose sort has every workgroup add up the counts of all others: here they are some hundred gigabytes of L2.
int check_gradient_tokens(const char* what, uint64_t n_tokens) {
  if (n_tokens > 1ull << 26) return fail(ETHA_ERR_UNSUPPORTED, "%s: %llu tokens; at most 2^26", what, (unsigned long long)n_tokens);
  return ETHA_OK;
}

// Column blocks, chunk length and workspace of a gradient call: a rule on sizes alone.
struct GradPlan {
  uint32_t n_cols, chunk, n_chunks;
  int passes, bits;
  uint32_t sort_blocks;
  uint64_t keys_bytes, hist_bytes, partial_bytes;
  uint64_t total() const { return 4 * keys_bytes + hist_bytes + partial_bytes; }
};
GradPlan grad_plan(uint64_t n, uint64_t n_rows, uint64_t width, int es) {
  GradPlan p = {};
  const uint64_t per = 64 * (16 / es);
  p.n_cols = (uint32_t)((width + per - 1) / per);
  // chunks of 128 places, shorter while there would be fewer waves than the chip holds a few of per SIMD, longer where the
  // pieces of rows that cross chunks would need more than 2048 places in the workspace
  uint64_t chunk = 128;
  while (chunk > 32 && (n + chunk - 1) / chunk * p.n_cols < 4096) chunk >>= 1;
  if ((n + chunk - 1) / chunk > 2048 && chunk == 128) chunk = ((n + 2047) / 2048 + 127) / 128 * 128;
  p.chunk = (uint32_t)chunk;
  p.n_chunks = (uint32_t)((n + chunk - 1) / chunk);
  const int bits = log2_up(n_rows + 1);
  p.passes = bits ? (bits + 8) / 9 : 1;
  p.bits = bits ? (bits + p.passes - 1) / p.passes : 1;
  p.sort_blocks = n <= kOneBlockTokens ? 0 : (uint32_t)((n + sort_tokens(n) - 1) / sort_tokens(n));
  const auto up = [](uint64_t b) { return (b + 255) / 256 * 256; };
  p.keys_bytes = up(n * 4);
  p.hist_bytes = up((uint64_t)p.sort_blocks * (1u << p.bits) * 4);
  p.partial_bytes = up((uint64_t)p.n_chunks * 2 * width * 4);
  return p;
}

int quantize_launch(const QuantArgs& a, uint32_t dtype, hipStream_t stream) {
  with_type(dtype, [&](auto s) {
    typedef decltype(s) S;
    // a wave (16 lanes for the narrowest: 45913 rows of 102 in bf16 6 us, 36 us with a wave) a row while the row fits its
    // registers, else a workgroup a row, with no more registers than the row needs (64128 rows of 4096 in fp32: 219 us with
    // room for 4096, 236 us with room for 8192)
    if (a.width <= 16 * 8 * 4)
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 16, 4>), dim3((uint32_t)((a.rows + 15) / 16)), dim3(256), 0, stream, a);
    else if (a.width <= 64 * 8 * 2)
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 64, 2>), dim3((uint32_t)((a.rows + 3) / 4)), dim3(256), 0, stream, a);
    else if (a.width <= 64 * 8 * 4)
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 64, 4>), dim3((uint32_t)((a.rows + 3) / 4)), dim3(256), 0, stream, a);
    else if (a.width <= 256 * 8 * 2)
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 256, 2>), dim3((uint32_t)a.rows), dim3(256), 0, stream, a);
    else if (a.width <= 256 * 8 * 4)
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 256, 4>), dim3((uint32_t)a.rows), dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((etha_quantize_rows_kernel<S, 1024, 4>), dim3((uint32_t)a.rows), dim3(1024), 0, stream, a);
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
  if (rc == ETHA_OK) rc = check_gradient_tokens("etha_embedding_grad_workspace", n_tokens);
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
  if (rc == ETHA_OK) rc = check_gradient_tokens("etha_embedding_grad", n_tokens);
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
    const dim3 grid((uint32_t)((n_rows + kGradWaves * kFewTokenRows - 1) / (kGradWaves * kFewTokenRows)), (uint32_t)((width + per - 1) / per));
    if (grid.x >= 1u << 24 || grid.y > 65535) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: too many rows or columns");
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
    uint32_t* keys[2] = {(uint32_t*)workspace, (uint32_t*)((char*)workspace + p.keys_bytes)};
    uint32_t* pos[2] = {(uint32_t*)((char*)workspace + 2 * p.keys_bytes), (uint32_t*)((char*)workspace + 3 * p.keys_bytes)};
    int at = 0;
    if (!p.sort_blocks) {
      hipLaunchKernelGGL(etha_sort_tokens_kernel, dim3(1), dim3(kOneBlockThreads), 0, (hipStream_t)stream, tokens,
                         (uint32_t)(token_dtype == ETHA_I64), (uint32_t)n_tokens, first_row, (uint32_t)n_rows, p.passes, p.bits,
                         keys[0], pos[0]);
      if ((rc = launched("etha_sort_tokens_kernel")) != ETHA_OK) return rc;
    } else {
      SortArgs s = {};
      s.tokens = tokens;
      s.wide = token_dtype == ETHA_I64;
      s.n = n_tokens;
      s.first = first_row;
      s.n_rows = (uint32_t)n_rows;
      s.bits = p.bits;
      s.hist = (uint32_t*)((char*)workspace + 4 * p.keys_bytes);
      for (int pass = 0; pass < p.passes; pass++) {
        s.shift = pass * p.bits;
        s.keys_in = pass ? keys[at ^ 1] : nullptr;
        s.pos_in = pass ? pos[at ^ 1] : nullptr;
        s.keys_out = keys[at];
        s.pos_out = pos[at];
        const bool wide_blocks = sort_tokens(n_tokens) == 4096;
        const auto count = wide_blocks ? etha_sort_count_kernel<4096> : etha_sort_count_kernel<1024>;
        const auto scatter = wide_blocks ? etha_sort_scatter_kernel<4096> : etha_sort_scatter_kernel<1024>;
        hipLaunchKernelGGL(count, dim3(p.sort_blocks), dim3(kSortThreads), 0, (hipStream_t)stream, s);
        if ((rc = launched("etha_sort_count_kernel")) != ETHA_OK) return rc;
        hipLaunchKernelGGL(scatter, dim3(p.sort_blocks), dim3(kSortThreads), 0, (hipStream_t)stream, s);
        if ((rc = launched("etha_sort_scatter_kernel")) != ETHA_OK) return rc;
        at ^= 1;
      }
      at ^= 1;
    }
    g.keys = keys[at];
    g.pos = pos[at];
    g.partial = (float*)((char*)workspace + 4 * p.keys_bytes + p.hist_bytes);
    g.chunk = p.chunk;
    g.n_chunks = p.n_chunks;
    g.n_cols = p.n_cols;
    const uint64_t blocks = ((uint64_t)p.n_chunks * p.n_cols + kGradWaves - 1) / kGradWaves;
    if (blocks > 1u << 23) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: too many tokens for this width");
    g.sum_blocks = (uint32_t)blocks;
  }
  const uint64_t zero_blocks = accumulate ? 0 : (n_rows + kZeroRows - 1) / kZeroRows;
  if (g.sum_blocks + zero_blocks >= 1u << 24) return fail(ETHA_ERR_UNSUPPORTED, "etha_embedding_grad: too many rows");
  with_type(grad_dtype, [&](auto s) {
    with_type(out_dtype, [&](auto d) {
      hipLaunchKernelGGL((etha_embedding_grad_kernel<decltype(s), decltype(d)>), dim3((uint32_t)(g.sum_blocks + zero_blocks)),
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
