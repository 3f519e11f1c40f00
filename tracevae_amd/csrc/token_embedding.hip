// Rows of a table by token id, times a scale, and the gradient of the table by sorted tokens.
//
//   out[r] = round(scale * W[ids[r]]),       zero rows for ids outside [0, V) and for the padding id
//   dW[v]  = round(scale * sum over r with ids[r] = v, in the order of r, of dout[r])
//
// Forward: a gather, bound by the bytes of the rows read and written.
//
// Gradient: the rows are brought into the order of their tokens by a stable counting sort of
// (token, row), then the sorted list is cut into tiles of equal length, whatever the frequencies are:
// a token that takes most of the list costs no more than many rare ones.  A group of lanes walks a
// tile for a slab of columns and writes every token that begins and ends inside it; the sums of a
// token that crosses tile borders go to a workspace and are joined in tile order.  Sums are fp32, in
// a fixed order, rounded once; no atomics on floats, so results repeat bit for bit.
#include "tv_common.h"

namespace {

constexpr int TE_THREADS = 256;
constexpr int TE_ITEMS = 2048;                    // ids per workgroup of a sort pass
constexpr int TE_MAX_BITS = 10;                   // of a digit
constexpr int TE_MAX_BINS = 1 << TE_MAX_BITS;

template <int N, typename T> struct Vec {
  T v[N];
} __attribute__((packed, aligned(sizeof(T))));

// N consecutive elements as floats; 16 bytes at once, at any alignment of the type
template <int N, typename T> __device__ __forceinline__ void load_n(const T *p, float (&x)[N]) {
  const Vec<N, T> f = *reinterpret_cast<const Vec<N, T> *>(p);
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = (float)f.v[j];
}
template <int N, typename T> __device__ __forceinline__ void store_n(T *p, const float (&x)[N]) {
  Vec<N, T> f;
#pragma unroll
  for (int j = 0; j < N; ++j) f.v[j] = (T)x[j];
  *reinterpret_cast<Vec<N, T> *>(p) = f;
}

// the part of a row that starts at column `col`: N columns, fewer at the end of the row
template <int N, typename T>
__device__ __forceinline__ void load_part(const T *row, int64_t col, int64_t dim, float (&x)[N]) {
  if (col + N <= dim) {
    load_n<N, T>(row + col, x);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = col + j < dim ? (float)row[col + j] : 0.f;
  }
}
template <int N, typename T>
__device__ __forceinline__ void store_part(T *row, int64_t col, int64_t dim, const float (&x)[N]) {
  if (col + N <= dim) {
    store_n<N, T>(row + col, x);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (col + j < dim) row[col + j] = (T)x[j];
  }
}

// ---------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------
template <typename W, typename O, int N>
__global__ __launch_bounds__(TE_THREADS) void lookup_kernel(int64_t rows, int64_t dim, int64_t vocab,
                                                            int64_t parts, const W *__restrict__ weight,
                                                            int64_t weight_stride,
                                                            const int64_t *__restrict__ ids,
                                                            int64_t padding, float scale,
                                                            O *__restrict__ out, int64_t out_stride) {
  const int64_t total = rows * parts, stride = (int64_t)gridDim.x * TE_THREADS;
  for (int64_t e = (int64_t)blockIdx.x * TE_THREADS + threadIdx.x; e < total; e += stride) {
    const int64_t r = e / parts, col = (e - r * parts) * N;
    const int64_t id = ids[r];
    float x[N];
    if (id >= 0 && id < vocab && id != padding) {
      load_part<N, W>(weight + id * weight_stride, col, dim, x);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = 0.f;
    }
    store_part<N, O>(out + r * out_stride, col, dim, x);
  }
}

// ---------------------------------------------------------------------------------------
// sort: one pass over one digit of the token = histogram, scan, scatter
// ---------------------------------------------------------------------------------------
// padding and ids outside the table get the token `vocab`, which sorts behind all others
__device__ __forceinline__ uint32_t token_of(int64_t id, int64_t vocab, int64_t padding) {
  return id >= 0 && id < vocab && id != padding ? (uint32_t)id : (uint32_t)vocab;
}
struct Keys {                                     // either the ids themselves or sorted pairs
  const int64_t *ids;
  const uint2 *pairs;
  int64_t vocab, padding;
  __device__ __forceinline__ uint2 at(int64_t i) const {
    return pairs ? pairs[i] : make_uint2(token_of(ids[i], vocab, padding), (uint32_t)i);
  }
};

__global__ __launch_bounds__(TE_THREADS) void digit_count_kernel(int64_t n, Keys keys, int shift,
                                                                 int bins, int64_t nblk,
                                                                 uint32_t *__restrict__ counts) {
  __shared__ uint32_t hist[TE_MAX_BINS];
  for (int b = threadIdx.x; b < bins; b += TE_THREADS) hist[b] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * TE_ITEMS;
  for (int k = threadIdx.x; k < TE_ITEMS; k += TE_THREADS)
    if (i0 + k < n) atomicAdd(&hist[(keys.at(i0 + k).x >> shift) & (bins - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += TE_THREADS) counts[(int64_t)b * nblk + blockIdx.x] = hist[b];
}

// per digit: counts -> exclusive sums over the workgroups, the total behind
__global__ __launch_bounds__(TE_THREADS) void digit_scan_kernel(int bins, int64_t nblk,
                                                                uint32_t *__restrict__ counts,
                                                                uint32_t *__restrict__ totals) {
  const int lane = threadIdx.x & 63;
  const int b = (int)blockIdx.x * (TE_THREADS / 64) + (threadIdx.x >> 6);
  if (b >= bins) return;
  uint32_t *row = counts + (int64_t)b * nblk;
  uint32_t carry = 0;
  for (int64_t i0 = 0; i0 < nblk; i0 += 64) {
    const uint32_t c = i0 + lane < nblk ? row[i0 + lane] : 0u;
    uint32_t s = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(s, o, 64);
      if (lane >= o) s += t;
    }
    if (i0 + lane < nblk) row[i0 + lane] = carry + s - c;
    carry += __shfl(s, 63, 64);
  }
  if (lane == 0) totals[b] = carry;
}

// stable: wave w of a workgroup takes the w-th quarter of its ids, 64 at a time; equal digits among
// the 64 are ranked by lane, and a wave's own counter carries the rank from round to round
__global__ __launch_bounds__(TE_THREADS) void digit_scatter_kernel(
    int64_t n, Keys keys, int shift, int bits, int64_t nblk, const uint32_t *__restrict__ counts,
    const uint32_t *__restrict__ totals, uint2 *__restrict__ out) {
  constexpr int WAVES = TE_THREADS / 64, ROUNDS = TE_ITEMS / TE_THREADS;
  __shared__ uint32_t seen[WAVES][TE_MAX_BINS];
  __shared__ uint32_t first[TE_MAX_BINS];
  __shared__ uint32_t wave_sum[WAVES];
  const int bins = 1 << bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int b = lane; b < bins; b += 64) seen[w][b] = 0;
  // first place of each digit: exclusive sums of the totals (4 digits per thread)
  {
    uint32_t c[TE_MAX_BINS / TE_THREADS], sum = 0;
#pragma unroll
    for (int k = 0; k < TE_MAX_BINS / TE_THREADS; ++k) {
      const int b = (int)threadIdx.x * (TE_MAX_BINS / TE_THREADS) + k;
      c[k] = b < bins ? totals[b] : 0u;
      sum += c[k];
    }
    uint32_t s = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(s, o, 64);
      if (lane >= o) s += t;
    }
    if (lane == 63) wave_sum[w] = s;
    __syncthreads();
    uint32_t before = s - sum;
    for (int k = 0; k < w; ++k) before += wave_sum[k];
#pragma unroll
    for (int k = 0; k < TE_MAX_BINS / TE_THREADS; ++k) {
      const int b = (int)threadIdx.x * (TE_MAX_BINS / TE_THREADS) + k;
      if (b < bins) first[b] = before + counts[(int64_t)b * nblk + blockIdx.x];
      before += c[k];
    }
  }
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * TE_ITEMS + (int64_t)w * (TE_ITEMS / WAVES);
  uint2 item[ROUNDS];
  uint32_t rank[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = i0 + k * 64 + lane;
    const bool in = i < n;
    item[k] = in ? keys.at(i) : make_uint2(0u, 0u);
    const uint32_t d = (item[k].x >> shift) & (bins - 1);
    uint64_t same = __ballot(in);
    for (int bit = 0; bit < bits; ++bit) {
      const uint64_t set = __ballot((d >> bit) & 1u);
      same &= (d >> bit) & 1u ? set : ~set;
    }
    const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
    rank[k] = 0;
    if (in) rank[k] = seen[w][d] + below;
    // (LDS accesses of one wave stay in order; the fences keep the compiler from moving them)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && below == 0) seen[w][d] += (uint32_t)__popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  __syncthreads();
  // where each wave's run of a digit begins
  for (int b = threadIdx.x; b < bins; b += TE_THREADS) {
    uint32_t at = first[b];
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const uint32_t c = seen[k][b];
      seen[k][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    const int64_t i = i0 + k * 64 + lane;
    if (i < n) out[seen[w][(item[k].x >> shift) & (bins - 1)] + rank[k]] = item[k];
  }
}

// ---------------------------------------------------------------------------------------
// sums over the sorted list
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(TE_THREADS) void zero_rows_kernel(int64_t n, T *__restrict__ x) {
  const int64_t stride = (int64_t)gridDim.x * TE_THREADS;
  for (int64_t i = (int64_t)blockIdx.x * TE_THREADS + threadIdx.x; i < n; i += stride) x[i] = (T)0.f;
}

// A group of G lanes, N columns each, walks one tile.  A token that neither begins before the tile
// nor goes on behind it is written to dW; the sum of one that began before goes to slot 0 of the
// tile, of one that begins here and goes on to slot 1.
template <typename D, typename W, int N, int G>
__global__ __launch_bounds__(TE_THREADS) void tile_sums_kernel(
    int64_t n, int64_t dim, int64_t vocab, int tile, int64_t tiles, int64_t slabs,
    const uint2 *__restrict__ sorted, const D *__restrict__ dout, int64_t dout_stride, float scale,
    W *__restrict__ dweight, float *__restrict__ part) {
  const int64_t unit = ((int64_t)blockIdx.x * TE_THREADS + threadIdx.x) / G;
  const int lane = threadIdx.x % G;
  if (unit >= tiles * slabs) return;
  const int64_t t = unit / slabs, col = ((unit - t * slabs) * G + lane) * N;
  const int64_t i0 = t * tile, i1 = i0 + tile < n ? i0 + tile : n;
  uint32_t cur = sorted[i0].x;
  if (cur >= vocab) return;                       // nothing but padding from here on
  bool began_before = i0 > 0 && sorted[i0 - 1].x == cur;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  auto write = [&](bool goes_on) {
    if (began_before || goes_on) {
      if (col < dim) store_part<N, float>(part + (t * 2 + (began_before ? 0 : 1)) * dim, col, dim, acc);
    } else {
      float y[N];
#pragma unroll
      for (int j = 0; j < N; ++j) y[j] = acc[j] * scale;
      if (col < dim) store_part<N, W>(dweight + (int64_t)cur * dim, col, dim, y);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    began_before = false;
  };
  for (int64_t i = i0; i < i1; ++i) {
    const uint2 p = sorted[i];
    if (p.x != cur) {
      write(false);
      cur = p.x;
      if (cur >= vocab) return;
    }
    float x[N];
    if (col < dim) {
      load_part<N, D>(dout + (int64_t)p.y * dout_stride, col, dim, x);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += x[j];
    }
  }
  write(i1 < n && sorted[i1].x == cur);
}

// the token that begins in tile t and goes on behind it: its slot there, then slot 0 of the tiles
// that follow, in order
template <typename W, int N, int G>
__global__ __launch_bounds__(TE_THREADS) void join_kernel(int64_t n, int64_t dim, int64_t vocab, int tile,
                                                          int64_t tiles, int64_t slabs,
                                                          const uint2 *__restrict__ sorted, float scale,
                                                          W *__restrict__ dweight,
                                                          const float *__restrict__ part) {
  const int64_t unit = ((int64_t)blockIdx.x * TE_THREADS + threadIdx.x) / G;
  const int lane = threadIdx.x % G;
  if (unit >= tiles * slabs) return;
  const int64_t t = unit / slabs, col = ((unit - t * slabs) * G + lane) * N;
  const int64_t i0 = t * tile, i1 = i0 + tile;
  if (i1 >= n || col >= dim) return;
  const uint32_t cur = sorted[i1 - 1].x;
  if (cur >= vocab || sorted[i1].x != cur) return;
  if (sorted[i0].x == cur && i0 > 0 && sorted[i0 - 1].x == cur) return;     // began before
  float acc[N];
  load_part<N, float>(part + (t * 2 + 1) * dim, col, dim, acc);
  for (int64_t u = t + 1; u < tiles && sorted[u * tile].x == cur; ++u) {
    float x[N];
    load_part<N, float>(part + u * 2 * dim, col, dim, x);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += x[j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] *= scale;
  store_part<N, W>(dweight + (int64_t)cur * dim, col, dim, acc);
}

// ---------------------------------------------------------------------------------------
struct Shape {
  int64_t nblk, tile, tiles;
  int passes, bits;
  int64_t pairs0, pairs1, counts, totals, part, bytes;
};
inline int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

inline Shape shape_of(int64_t rows, int64_t dim, int64_t vocab) {
  Shape s = {};
  s.nblk = tv_cdiv(rows, TE_ITEMS);
  int bits = 1;
  while (bits < 32 && ((int64_t)1 << bits) < vocab + 1) ++bits;
  s.passes = (int)tv_cdiv(bits, TE_MAX_BITS);
  s.bits = (int)tv_cdiv(bits, s.passes);
  s.tile = 32;
  s.tiles = tv_cdiv(rows, s.tile);
  s.pairs0 = 0;
  s.pairs1 = align256(rows * 8);
  s.counts = s.pairs1 + (s.passes > 1 ? align256(rows * 8) : 0);
  s.totals = s.counts + align256(s.nblk * ((int64_t)4 << s.bits));
  s.part = s.totals + align256((int64_t)4 << s.bits);
  s.bytes = s.part + align256(s.tiles * 2 * dim * 4);
  return s;
}

inline bool sizes_ok(int64_t rows, int64_t dim, int64_t vocab) {
  // (so that sorted positions and tokens fit 32 bits, and tiles * slabs a grid)
  return rows >= 0 && rows < INT32_MAX && dim >= 1 && dim <= (1 << 16) && vocab >= 1 && vocab < INT32_MAX;
}

template <typename W, typename O>
void launch_lookup(int64_t rows, int64_t dim, int64_t vocab, const void *weight, int64_t weight_stride,
                   const int64_t *ids, int64_t padding, float scale, void *out, int64_t out_stride,
                   hipStream_t stream) {
  constexpr int N = 16 / (sizeof(W) < sizeof(O) ? sizeof(O) : sizeof(W));
  const int64_t parts = tv_cdiv(dim, N);
  int64_t blocks = tv_cdiv(rows * parts, TE_THREADS);
  if (blocks > 16384) blocks = 16384;
  hipLaunchKernelGGL((lookup_kernel<W, O, N>), dim3((unsigned)blocks), dim3(TE_THREADS), 0, stream, rows,
                     dim, vocab, parts, (const W *)weight, weight_stride, ids, padding, scale, (O *)out,
                     out_stride);
}

template <typename D, typename W>
void launch_sums(const Shape &s, int64_t rows, int64_t dim, int64_t vocab, const uint2 *sorted,
                 const void *dout, int64_t dout_stride, float scale, void *dweight, float *part,
                 hipStream_t stream) {
  constexpr int N = 16 / sizeof(D), G = 64;
  const int64_t slabs = tv_cdiv(dim, N * G);
  const unsigned blocks = (unsigned)tv_cdiv(s.tiles * slabs * G, TE_THREADS);
  hipLaunchKernelGGL((tile_sums_kernel<D, W, N, G>), dim3(blocks), dim3(TE_THREADS), 0, stream, rows, dim,
                     vocab, (int)s.tile, s.tiles, slabs, sorted, (const D *)dout, dout_stride, scale,
                     (W *)dweight, part);
  hipLaunchKernelGGL((join_kernel<W, N, G>), dim3(blocks), dim3(TE_THREADS), 0, stream, rows, dim, vocab,
                     (int)s.tile, s.tiles, slabs, sorted, scale, (W *)dweight, part);
}

// (table, rows) types: equal, or an fp32 table with 16-bit rows
inline bool types_ok(int table, int rows) {
  return table >= TV_DTYPE_F32 && table <= TV_DTYPE_F16 && rows >= TV_DTYPE_F32 && rows <= TV_DTYPE_F16 &&
         (table == rows || table == TV_DTYPE_F32);
}
inline int64_t width_of(int dtype) { return dtype == TV_DTYPE_F32 ? 4 : 2; }

}  // namespace

extern "C" int tv_scaled_embedding_fwd(int64_t rows, int64_t dim, int64_t num_tokens, int weight_dtype,
                                       int out_dtype, const void *weight, int64_t weight_stride,
                                       const int64_t *ids, int64_t padding_id, float scale, void *out,
                                       int64_t out_stride, void *stream) {
  TV_REQUIRE(sizes_ok(rows, dim, num_tokens), "tv_scaled_embedding_fwd: bad sizes");
  TV_REQUIRE(types_ok(weight_dtype, out_dtype),
             "tv_scaled_embedding_fwd: the rows have the table's type, or 16 bits of an fp32 table");
  TV_REQUIRE(weight_stride >= dim && out_stride >= dim, "tv_scaled_embedding_fwd: rows overlap");
  if (rows == 0) return TV_OK;
  TV_REQUIRE(weight && ids && out, "tv_scaled_embedding_fwd: null pointer");
  TV_REQUIRE(((uintptr_t)weight & (uintptr_t)(width_of(weight_dtype) - 1)) == 0 &&
                 ((uintptr_t)out & (uintptr_t)(width_of(out_dtype) - 1)) == 0 && ((uintptr_t)ids & 7) == 0,
             "tv_scaled_embedding_fwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
#define TE_GO(W, O) \
  launch_lookup<W, O>(rows, dim, num_tokens, weight, weight_stride, ids, padding_id, scale, out, out_stride, st)
  if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_F32) TE_GO(float, float);
  else if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_BF16) TE_GO(float, __bf16);
  else if (weight_dtype == TV_DTYPE_F32) TE_GO(float, _Float16);
  else if (weight_dtype == TV_DTYPE_BF16) TE_GO(__bf16, __bf16);
  else TE_GO(_Float16, _Float16);
#undef TE_GO
  TV_LAUNCH_CHECK("tv_scaled_embedding_fwd");
  return TV_OK;
}

extern "C" int64_t tv_scaled_embedding_bwd_workspace_bytes(int64_t rows, int64_t dim, int64_t num_tokens) {
  if (!sizes_ok(rows, dim, num_tokens)) return -1;
  return rows == 0 ? 0 : shape_of(rows, dim, num_tokens).bytes;
}

extern "C" int tv_scaled_embedding_bwd(int64_t rows, int64_t dim, int64_t num_tokens, int weight_dtype,
                                       int out_dtype, const int64_t *ids, int64_t padding_id, float scale,
                                       const void *dout, int64_t dout_stride, void *dweight,
                                       void *workspace, int64_t workspace_bytes, void *stream) {
  TV_REQUIRE(sizes_ok(rows, dim, num_tokens), "tv_scaled_embedding_bwd: bad sizes");
  TV_REQUIRE(types_ok(weight_dtype, out_dtype),
             "tv_scaled_embedding_bwd: the rows have the table's type, or 16 bits of an fp32 table");
  TV_REQUIRE(dweight && (rows == 0 || (ids && dout)), "tv_scaled_embedding_bwd: null pointer");
  TV_REQUIRE(rows == 0 || dout_stride >= dim, "tv_scaled_embedding_bwd: rows overlap");
  TV_REQUIRE(((uintptr_t)dweight & (uintptr_t)(width_of(weight_dtype) - 1)) == 0 &&
                 ((uintptr_t)dout & (uintptr_t)(width_of(out_dtype) - 1)) == 0 && ((uintptr_t)ids & 7) == 0 &&
                 ((uintptr_t)workspace & 15) == 0,
             "tv_scaled_embedding_bwd: misaligned pointer");
  hipStream_t st = (hipStream_t)stream;
  const Shape s = shape_of(rows, dim, num_tokens);
  if (rows > 0) {
    TV_REQUIRE(workspace, "tv_scaled_embedding_bwd: null workspace");
    if (workspace_bytes < s.bytes) {
      tv_set_error("tv_scaled_embedding_bwd: workspace too small");
      return TV_ERR_WORKSPACE;
    }
  }
  {
    const int64_t count = num_tokens * dim;
    int64_t blocks = tv_cdiv(count, TE_THREADS * 8);
    if (blocks > 16384) blocks = 16384;
    if (weight_dtype == TV_DTYPE_F32)
      hipLaunchKernelGGL(zero_rows_kernel<float>, dim3((unsigned)blocks), dim3(TE_THREADS), 0, st, count,
                         (float *)dweight);
    else
      hipLaunchKernelGGL(zero_rows_kernel<_Float16>, dim3((unsigned)blocks), dim3(TE_THREADS), 0, st, count,
                         (_Float16 *)dweight);
    TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
  }
  if (rows == 0) return TV_OK;
  char *ws = (char *)workspace;
  uint2 *pairs[2] = {(uint2 *)(ws + s.pairs0), (uint2 *)(ws + s.pairs1)};
  uint32_t *counts = (uint32_t *)(ws + s.counts), *totals = (uint32_t *)(ws + s.totals);
  Keys keys = {ids, nullptr, num_tokens, padding_id};
  for (int p = 0; p < s.passes; ++p) {
    uint2 *to = pairs[(s.passes - 1 - p) & 1];    // (the last pass writes pairs[0])
    const int bins = 1 << s.bits;
    hipLaunchKernelGGL(digit_count_kernel, dim3((unsigned)s.nblk), dim3(TE_THREADS), 0, st, rows, keys,
                       p * s.bits, bins, s.nblk, counts);
    hipLaunchKernelGGL(digit_scan_kernel, dim3((unsigned)tv_cdiv(bins, TE_THREADS / 64)), dim3(TE_THREADS), 0,
                       st, bins, s.nblk, counts, totals);
    hipLaunchKernelGGL(digit_scatter_kernel, dim3((unsigned)s.nblk), dim3(TE_THREADS), 0, st, rows, keys,
                       p * s.bits, s.bits, s.nblk, counts, totals, to);
    TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
    keys.pairs = to;
  }
  float *part = (float *)(ws + s.part);
#define TE_GO(D, W) launch_sums<D, W>(s, rows, dim, num_tokens, pairs[0], dout, dout_stride, scale, dweight, part, st)
  if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_F32) TE_GO(float, float);
  else if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_BF16) TE_GO(__bf16, float);
  else if (weight_dtype == TV_DTYPE_F32) TE_GO(_Float16, float);
  else if (weight_dtype == TV_DTYPE_BF16) TE_GO(__bf16, __bf16);
  else TE_GO(_Float16, _Float16);
#undef TE_GO
  TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
  return TV_OK;
}
