// Rows of a table by token id, times a scale, and the gradient of the table by sorted tokens.
//
//   out[r] = round(fp32(scale * W[ids[r]])), zero rows for ids outside [0, V) and for the padding id
//   dW[v]  = round(scale * sum over r with ids[r] = v, in the order of r, of dout[r])
//
// Forward: a gather, bound by the bytes of the rows read and written.
//
// Gradient: the rows are brought into the order of their tokens by a stable counting sort of
// (token, row), then the sorted list is cut into tiles of equal length, whatever the frequencies are:
// a token that takes most of the list costs no more than many rare ones.  A group of lanes walks a
// tile for a slab of columns and writes every token that begins and ends inside it; the sums of a
// token that crosses tile borders go to a workspace and are joined in tile order.  Sums are fp32, in
// a fixed order, the product with the scale too, then rounded to the type; no atomics on floats, so
// results repeat bit for bit.
//
// Measured (kernels alone): lookup of 65536 x 4096 bf16 116 us (837 MB read and written,
// 7.2 TB/s).  Gradient of 262144 x 512 bf16 over 1000 tokens, half of the rows on three of
// them: sort 5 + 13, tiles 49 (268 MB read, 5.5 TB/s), join 15 us.  Of 32768 x 1024 bf16 into 50001 fp32
// rows: sort 18, tiles and zero rows 46 (269 MB, 5.8 TB/s), join 9.  Of 25600 x 40 fp32 over 1000: sort 3
// + 7, tiles 6, join 13; of 1021 x 251 fp16: sort 6, tiles 6, join 6 - a chain of dependent loads each.
#include "tv_common.h"

namespace {

constexpr int TE_THREADS = 256;
constexpr int TE_LOOKUP_THREADS = 512;
constexpr int TE_SORT_THREADS = 1024;             // of a sort workgroup
constexpr int TE_SORT_WAVES = TE_SORT_THREADS / 64;
constexpr int TE_TINY = 128;                      // rows whose gradient is one launch
constexpr int TE_SMALL = 8192;                    // rows that one workgroup sorts alone
constexpr int TE_SORT_BLOCKS = 64;                // sort workgroups of longer lists, at most
constexpr int TE_MAX_BITS = 10;                   // of a digit
constexpr int TE_MAX_BINS = 1 << TE_MAX_BITS;
constexpr int TE_BATCH = 8;                       // rows whose loads are in flight together
constexpr int TE_JOIN_THREADS = 1024;
constexpr int TE_LONG = 16;                       // tiles of a token that one group joins alone

// N consecutive elements at any alignment of the type, in one access of up to 16 bytes
template <int N, typename T> struct Some {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V Any __attribute__((aligned(sizeof(T))));
};
template <int N, typename T, bool PAST = false> __device__ __forceinline__ void load_n(const T *p, float (&x)[N]) {
  constexpr int M = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
  if constexpr (N == 1) {
    x[0] = (float)p[0];
  } else {
#pragma unroll
    for (int k = 0; k < N; k += M) {
      typedef typename Some<M, T>::Any Any;
      const Any *q = reinterpret_cast<const Any *>(p + k);
      const typename Some<M, T>::V f = PAST ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int j = 0; j < M; ++j) x[k + j] = (float)f[j];
    }
  }
}
template <int N, typename T, bool PAST = false> __device__ __forceinline__ void store_n(T *p, const float (&x)[N]) {
  constexpr int M = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
  if constexpr (N == 1) {
    p[0] = (T)x[0];
  } else {
#pragma unroll
    for (int k = 0; k < N; k += M) {
      typedef typename Some<M, T>::Any Any;
      typename Some<M, T>::V f;
#pragma unroll
      for (int j = 0; j < M; ++j) f[j] = (T)x[k + j];
      if (PAST) __builtin_nontemporal_store(f, reinterpret_cast<Any *>(p + k));
      else *reinterpret_cast<Any *>(p + k) = f;
    }
  }
}

// Columns of a row are cut into parts of N; the last part ends with the row and overlaps the one in
// front of it if N does not divide the row: both hold the same values there, so no part is masked.
// Rows shorter than N use N = 1.
__device__ __forceinline__ int64_t part_column(int64_t part, int n, int64_t dim) {
  const int64_t c = part * n;
  return c + n <= dim ? c : dim - n;
}

// ---------------------------------------------------------------------------------------
// Forward: 2^lg threads per row, ROWS rows per thread with their loads in flight together.  The rows are
// stored past the caches: a lookup of 64, 256 and 512 MiB takes 17, 62 and 133 us so and 18, 75 and 144
// without the hint, a lookup and one pass that reads its result 37, 132 and 252 against 35, 138 and 271 -
// and without it what follows pays for the dirty lines (lookup and gradient of 32768 x 1024: 92 us
// against 107).  512 threads and 2 rows each: 65536 x 4096 bf16 135 us (256 and 4: 143, 512 and 1: 173, 1024
// and 2: 142), 16384 x 4096 fp32 68 (83, 76, 65), 262144 x 512 bf16 40 (44, 73, 42).
// ---------------------------------------------------------------------------------------
template <typename W, typename O, int N, int ROWS>
__global__ __launch_bounds__(TE_LOOKUP_THREADS) void lookup_kernel(int64_t rows, int64_t dim, int64_t vocab,
                                                            int parts, int lg, const W *__restrict__ weight,
                                                            int64_t weight_stride,
                                                            const int64_t *__restrict__ ids,
                                                            int64_t padding, float scale,
                                                            O *__restrict__ out, int64_t out_stride) {
  const int per = TE_LOOKUP_THREADS >> lg;        // rows per workgroup and trip
  const int64_t r0 = (int64_t)blockIdx.x * per * ROWS + (threadIdx.x >> lg);
  int64_t id[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const int64_t r = r0 + (int64_t)k * per;
    id[k] = r < rows ? ids[r] : -1;
    if (id[k] >= vocab || id[k] == padding) id[k] = -1;
  }
  for (int part = threadIdx.x & ((1 << lg) - 1); part < parts; part += 1 << lg) {
    const int64_t col = part_column(part, N, dim);
    float x[ROWS][N];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      if (id[k] >= 0) {
        load_n<N, W>(weight + id[k] * weight_stride + col, x[k]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[k][j] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t r = r0 + (int64_t)k * per;
      if (r >= rows) break;
      if (id[k] >= 0) {                           // (0 * scale is no zero for an infinite scale)
#pragma unroll
        for (int j = 0; j < N; ++j) x[k][j] *= scale;
      }
      store_n<N, O, true>(out + r * out_stride + col, x[k]);
    }
  }
}

// ---------------------------------------------------------------------------------------
// stable counting sort of (token, row) by digits of the token, lowest first
// ---------------------------------------------------------------------------------------
// padding and ids outside the table get the token `vocab`, which sorts behind all others
__device__ __forceinline__ uint32_t token_of(int64_t id, int64_t vocab, int64_t padding) {
  return id >= 0 && id < vocab && id != padding ? (uint32_t)id : (uint32_t)vocab;
}
struct Keys {                                     // either the ids themselves or pairs of an earlier pass
  const int64_t *ids;
  const uint2 *pairs;
  int64_t vocab, padding;
  __device__ __forceinline__ uint2 at(int64_t i) const {
    return pairs ? pairs[i] : make_uint2(token_of(ids[i], vocab, padding), (uint32_t)i);
  }
};

// lanes of the wave with the same digit (among those that are `in`)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, bool in, int bits) {
  uint64_t same = __ballot(in);
  for (int bit = 0; bit < bits; ++bit) {
    const uint64_t set = __ballot((d >> bit) & 1u);
    same &= (d >> bit) & 1u ? set : ~set;
  }
  return same;
}
// exclusive sum over the 1024 threads of a sort workgroup
__device__ __forceinline__ uint32_t sort_exclusive_sum(uint32_t c, uint32_t *wave_sum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t s = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(s, o, 64);
    if (lane >= o) s += t;
  }
  if (lane == 63) wave_sum[w] = s;
  __syncthreads();
  uint32_t before = s - c;
  for (int k = 0; k < w; ++k) before += wave_sum[k];
  __syncthreads();
  return before;
}

// Up to TE_SMALL rows: all passes in one workgroup, the pairs in LDS between them (1021 rows: 6 us; the
// launches of the longer form take 10 at least).  Wave w takes the
// w-th run of 64 * ROUNDS pairs; equal digits among 64 are ranked by lane, and the wave's own counter
// carries the rank from round to round.
template <int ROUNDS>
__global__ __launch_bounds__(TE_SORT_THREADS) void small_sort_kernel(int n, Keys keys, int bits, int passes,
                                                                     uint2 *__restrict__ out) {
  __shared__ uint32_t seen[TE_SORT_WAVES][TE_MAX_BINS];
  __shared__ uint32_t wave_sum[TE_SORT_WAVES];
  __shared__ uint2 pairs[ROUNDS * TE_SORT_THREADS];
  const int bins = 1 << bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int i0 = w * 64 * ROUNDS + lane;
  uint2 item[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) item[k] = i0 + k * 64 < n ? keys.at(i0 + k * 64) : make_uint2(0u, 0u);
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    for (int b = lane; b < bins; b += 64) seen[w][b] = 0;
    uint32_t rank[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
      const bool in = i0 + k * 64 < n;
      const uint32_t d = (item[k].x >> shift) & (bins - 1);
      const uint64_t same = same_digit(d, in, bits);
      const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
      // (LDS accesses of one wave stay in order; the fences keep the compiler from moving them)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      rank[k] = in ? seen[w][d] + below : 0u;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (in && below == 0) seen[w][d] += (uint32_t)__popcll(same);
    }
    __syncthreads();
    // counts -> first places: digits in order, within a digit the waves in order
    uint32_t total = 0;
    const int b = threadIdx.x;
    if (b < bins) {
#pragma unroll
      for (int k = 0; k < TE_SORT_WAVES; ++k) {
        const uint32_t c = seen[k][b];
        seen[k][b] = total;
        total += c;
      }
    }
    const uint32_t first = sort_exclusive_sum(b < bins ? total : 0u, wave_sum);
    if (b < bins) {
#pragma unroll
      for (int k = 0; k < TE_SORT_WAVES; ++k) seen[k][b] += first;
    }
    __syncthreads();
    uint2 *to = p + 1 < passes ? pairs : out;
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
      if (i0 + k * 64 < n) to[seen[w][(item[k].x >> shift) & (bins - 1)] + rank[k]] = item[k];
    if (p + 1 < passes) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < ROUNDS; ++k)
        if (i0 + k * 64 < n) item[k] = pairs[i0 + k * 64];
    }
  }
}

// Longer lists: every workgroup takes one run of `items` (a multiple of 64 * TE_SORT_WAVES) pairs.
__global__ __launch_bounds__(TE_SORT_THREADS) void digit_count_kernel(int64_t n, Keys keys, int shift,
                                                                      int bits, int64_t items,
                                                                      uint32_t *__restrict__ counts) {
  __shared__ uint32_t hist[TE_MAX_BINS];
  const int bins = 1 << bits;
  if ((int)threadIdx.x < bins) hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * items, i1 = i0 + items < n ? i0 + items : n;
#pragma unroll 4
  for (int64_t i = i0 + threadIdx.x; i < i1; i += TE_SORT_THREADS)
    atomicAdd(&hist[(keys.at(i).x >> shift) & (bins - 1)], 1u);
  __syncthreads();
  if ((int)threadIdx.x < bins) counts[(int64_t)blockIdx.x * bins + threadIdx.x] = hist[threadIdx.x];
}

// KEEP: a wave's run has at most that many rounds of 64 pairs, which stay in registers
template <int KEEP>
__global__ __launch_bounds__(TE_SORT_THREADS) void digit_scatter_kernel(
    int64_t n, Keys keys, int shift, int bits, int64_t items, int nblk,
    const uint32_t *__restrict__ counts, uint2 *__restrict__ out) {
  __shared__ uint32_t seen[TE_SORT_WAVES][TE_MAX_BINS];
  __shared__ uint32_t wave_sum[TE_SORT_WAVES];
  const int bins = 1 << bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6, b = threadIdx.x;
  const int64_t run = items / TE_SORT_WAVES;
  const int64_t i0 = (int64_t)blockIdx.x * items + w * run;
  const int64_t i1 = i0 + run < n ? i0 + run : n;
  uint2 kept[KEEP > 0 ? KEEP : 1];
  if (KEEP > 0) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      kept[k] = i0 + k * 64 + lane < i1 ? keys.at(i0 + k * 64 + lane) : make_uint2(0u, 0u);
  }
  for (int k = lane; k < bins; k += 64) seen[w][k] = 0;
  // the digit's pairs in the workgroups before this one, and in all
  uint32_t before = 0, total = 0;
  if (b < bins) {
    for (int k0 = 0; k0 < nblk; k0 += 16) {
      uint32_t c[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) c[k] = k0 + k < nblk ? counts[(int64_t)(k0 + k) * bins + b] : 0u;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        before += k0 + k < (int)blockIdx.x ? c[k] : 0u;
        total += c[k];
      }
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  auto digit = [&](uint2 item) { return (item.x >> shift) & (bins - 1); };
  if (KEEP > 0) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k)
      if (i0 + k * 64 + lane < i1) atomicAdd(&seen[w][digit(kept[k])], 1u);
  } else {
    for (int64_t i = i0 + lane; i < i1; i += 64) atomicAdd(&seen[w][digit(keys.at(i))], 1u);
  }
  __syncthreads();
  uint32_t at = sort_exclusive_sum(b < bins ? total : 0u, wave_sum) + before;
  if (b < bins) {
#pragma unroll
    for (int k = 0; k < TE_SORT_WAVES; ++k) {
      const uint32_t c = seen[k][b];
      seen[k][b] = at;
      at += c;
    }
  }
  __syncthreads();
  auto place = [&](uint2 item, bool in) {
    const uint32_t d = digit(item);
    const uint64_t same = same_digit(d, in, bits);
    const uint32_t below = (uint32_t)__popcll(same & ((1ull << lane) - 1ull));
    // (LDS accesses of one wave stay in order; the fences keep the compiler from moving them)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint32_t to = in ? seen[w][d] + below : 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in && below == 0) seen[w][d] += (uint32_t)__popcll(same);
    if (in) out[to] = item;
  };
  if (KEEP > 0) {
#pragma unroll
    for (int k = 0; k < KEEP; ++k) place(kept[k], i0 + k * 64 + lane < i1);
  } else {
    for (int64_t j = i0; j < i1; j += 64) {
      const bool in = j + lane < i1;
      place(in ? keys.at(j + lane) : make_uint2(0u, 0u), in);
    }
  }
}

// ---------------------------------------------------------------------------------------
// sums over the sorted list
// ---------------------------------------------------------------------------------------
// Rows of dW that no token names, `each` (up to 16) per wave: a binary search in the sorted list for each.
// They are stored past the caches (50001 x 1024 fp32, three quarters of it zeros: 92 us for lookup and
// gradient against 101 without; the rows that hold sums lose by it).
template <typename W>
__device__ __forceinline__ void zero_absent_rows(int64_t wave, int each, int64_t n, int64_t dim, int64_t vocab,
                                                 const uint2 *__restrict__ sorted, W *__restrict__ dweight) {
  const int lane = threadIdx.x & 63;
  const int64_t v0 = wave * each, v = v0 + lane;
  bool absent = false;
  if (lane < each && v < vocab) {
    int64_t lo = 0, hi = n;                       // the first pair whose token is not below v
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if ((int64_t)sorted[mid].x < v) lo = mid + 1;
      else hi = mid;
    }
    absent = lo >= n || (int64_t)sorted[lo].x != v;
  }
  uint64_t rows = __ballot(absent);
  while (rows) {
    const int bit = __builtin_ctzll(rows);
    rows &= rows - 1;
    W *row = dweight + (v0 + bit) * dim;
    constexpr int M = 16 / sizeof(W);
    if (dim >= M) {
      const int64_t parts = (dim + M - 1) / M;
      for (int64_t part = lane; part < parts; part += 64) {
        float zero[M];
#pragma unroll
        for (int j = 0; j < M; ++j) zero[j] = 0.f;
        store_n<M, W, true>(row + part_column(part, M, dim), zero);
      }
    } else if (lane < dim) {
      row[lane] = (W)0.f;
    }
  }
}

// A group of G lanes, N columns each, walks one tile.  A token that neither begins before the tile
// nor goes on behind it is written to dW; the sum of one that began before goes to slot 0 of the
// tile, of one that begins here and goes on to slot 1.
template <typename D, typename W, int N, int G>
__global__ __launch_bounds__(TE_THREADS) void tile_sums_kernel(
    int64_t n, int64_t dim, int64_t vocab, int tile, int64_t tiles, int64_t slabs, int64_t tile_blocks,
    int zero_rows, const uint2 *__restrict__ sorted, const D *__restrict__ dout, int64_t dout_stride, float scale,
    W *__restrict__ dweight, float *__restrict__ part) {
  if ((int64_t)blockIdx.x >= tile_blocks) {
    zero_absent_rows<W>(((int64_t)blockIdx.x - tile_blocks) * (TE_THREADS / 64) + (threadIdx.x >> 6), zero_rows, n,
                        dim, vocab, sorted, dweight);
    return;
  }
  const int64_t unit = (int64_t)blockIdx.x * (TE_THREADS / G) + threadIdx.x / G;
  if (unit >= tiles * slabs) return;
  const int64_t t = unit / slabs, column_part = (unit - t * slabs) * G + threadIdx.x % G;
  const bool active = column_part * N < dim;
  const int64_t col = active ? part_column(column_part, N, dim) : 0;
  const int64_t i0 = t * tile, i1 = i0 + tile < n ? i0 + tile : n;
  uint32_t cur = sorted[i0].x;
  if (cur >= vocab) return;                       // nothing but padding from here on
  bool began_before = i0 > 0 && sorted[i0 - 1].x == cur;
  const uint32_t behind = i1 < n ? sorted[i1].x : 0xffffffffu;
  float acc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  auto write = [&](bool goes_on) {
    if (active) {
      if (began_before || goes_on) {
        store_n<N, float>(part + (t * 2 + (began_before ? 0 : 1)) * dim + col, acc);
      } else {
        float y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = acc[j] * scale;
        store_n<N, W>(dweight + (int64_t)cur * dim + col, y);
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    began_before = false;
  };
  uint2 next[TE_BATCH];
#pragma unroll
  for (int k = 0; k < TE_BATCH; ++k) next[k] = sorted[i0 + k < i1 ? i0 + k : i1 - 1];
  for (int64_t i = i0; i < i1; i += TE_BATCH) {
    uint2 p[TE_BATCH];
    float x[TE_BATCH][N];
#pragma unroll
    for (int k = 0; k < TE_BATCH; ++k) p[k] = next[k];
#pragma unroll
    for (int k = 0; k < TE_BATCH; ++k)            // (rows of padding are inside dout as well; read once)
      load_n<N, D, true>(dout + (int64_t)p[k].y * dout_stride + col, x[k]);
#pragma unroll
    for (int k = 0; k < TE_BATCH; ++k) {          // the next pairs, on their way behind these rows
      const int64_t q = i + TE_BATCH + k;
      next[k] = sorted[q < i1 ? q : i1 - 1];
    }
#pragma unroll
    for (int k = 0; k < TE_BATCH; ++k) {
      if (i + k >= i1) break;
      if (p[k].x != cur) {
        write(false);
        cur = p[k].x;
        if (cur >= vocab) return;
      }
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] += x[k][j];
    }
  }
  write(behind == cur);
}

// The token that begins in tile t and goes on behind it: its slot there, then slot 0 of the tiles
// that follow, in order.  A group of G lanes takes the token of one tile; one of more than TE_LONG
// tiles is left to the whole workgroup, whose groups take one run of its tiles each.  The slabs of a token
// are in different workgroups (32768 x 2048 fp32 over 1000 tokens 70 us against 86 with the slabs side by
// side, 65536 x 4096 bf16 over 32000 168 against 189): one CU reads no more than some 100 GB/s.
template <typename W, int N, int G>
__global__ __launch_bounds__(TE_JOIN_THREADS) void join_kernel(int64_t n, int64_t dim, int64_t vocab, int tile,
                                                               int64_t tiles, int64_t slabs,
                                                               const uint2 *__restrict__ sorted, float scale,
                                                               W *__restrict__ dweight,
                                                               const float *__restrict__ part) {
  constexpr int GROUPS = TE_JOIN_THREADS / G;
  __shared__ int64_t long_end[GROUPS];            // the tile behind the last one of a long token, or 0
  __shared__ float sums[GROUPS][G * N];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  auto tile_of = [&](int g, int64_t &t, int64_t &col) -> bool {
    const int64_t unit = (int64_t)blockIdx.x * GROUPS + g;
    const int64_t slab = unit / tiles;
    t = slab < slabs ? unit - slab * tiles : tiles;
    const int64_t column_part = slab * G + lane;
    const bool active = column_part * N < dim;
    col = active ? part_column(column_part, N, dim) : 0;
    return active;
  };
  // acc += slot 0 of the tiles u0 .. u1 - 1, in order
  auto add = [&](int64_t u0, int64_t u1, int64_t col, float (&acc)[N]) {
    for (int64_t u = u0; u < u1; u += TE_BATCH) {
      float x[TE_BATCH][N];
#pragma unroll
      for (int k = 0; k < TE_BATCH; ++k)
        load_n<N, float>(part + (u + k < u1 ? u + k : u1 - 1) * 2 * dim + col, x[k]);
#pragma unroll
      for (int k = 0; k < TE_BATCH; ++k) {
        if (u + k >= u1) break;
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += x[k][j];
      }
    }
  };
  int64_t t, col;
  const bool active = tile_of(group, t, col);
  if (lane == 0) long_end[group] = 0;
  const int64_t i0 = t * tile, i1 = i0 + tile;
  if (t < tiles && i1 < n) {
    const uint32_t cur = sorted[i1 - 1].x;
    const uint32_t next = sorted[i1].x, head = sorted[i0].x, prev = sorted[i0 > 0 ? i0 - 1 : 0].x;
    if (cur < vocab && next == cur && !(head == cur && i0 > 0 && prev == cur)) {
      // the first tile that does not begin with the token, by G probes at a time: first the next G tiles
      // (a token seldom has more), then G of the rest
      auto run_of = [&](int64_t probe, int64_t end) -> int {
        const uint64_t all = __ballot(probe < end && sorted[(probe < end ? probe : end - 1) * tile].x == cur);
        return __popcll(G == 64 ? all : (all >> ((threadIdx.x & 63) & ~(G - 1))) & ((1ull << (G & 63)) - 1ull));
      };
      int64_t lo = t + 1, hi = tiles;
      const int run = run_of(lo + lane, hi);
      if (run < G && run <= TE_LONG) {
        float acc[N];
        load_n<N, float>(part + (t * 2 + 1) * dim + col, acc);
        add(t + 1, t + 1 + run, col, acc);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] *= scale;
        if (active) store_n<N, W>(dweight + (int64_t)cur * dim + col, acc);
      } else {
        lo += run;
        while (run == G && lo < hi) {
          const int64_t step = (hi - lo + G - 1) / G;
          lo += run_of(lo + (lane + 1) * step - 1, hi) * step;
          hi = lo + step - 1 < hi ? lo + step - 1 : hi;
        }
        if (lane == 0) long_end[group] = lo;
      }
    }
  }
  __syncthreads();
  for (int g = 0; g < GROUPS; ++g) {
    const int64_t to = long_end[g];
    if (to == 0) continue;
    const bool on = tile_of(g, t, col);
    const int64_t count = to - (t + 1);
    const int64_t each = count > GROUPS * TE_BATCH ? (count + GROUPS - 1) / GROUPS : TE_BATCH;
    const int used = (int)((count + each - 1) / each);
    const int64_t u0 = t + 1 + group * each < to ? t + 1 + group * each : to;
    const int64_t u1 = u0 + each < to ? u0 + each : to;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    if (group == 0) load_n<N, float>(part + (t * 2 + 1) * dim + col, acc);
    if (group < used) {
      add(u0, u1, col, acc);
#pragma unroll
      for (int j = 0; j < N; ++j) sums[group][j * G + lane] = acc[j];
    }
    __syncthreads();
    if (group == 0) {
      for (int k = 1; k < used; ++k)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += sums[k][j * G + lane];
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] *= scale;
      if (on) store_n<N, W>(dweight + (int64_t)sorted[(t + 1) * tile].x * dim + col, acc);
    }
    __syncthreads();
  }
}

// Up to TE_TINY rows: no sort.  16 to 128 rows of 40 fp32 into 1000 table rows 4.4-5.3 us (sorted: 14.2-14.9), of
// 251 fp16 into 997 4.8-5.5 (12.4-14.6), of 64 fp32 into 50001 5.8-6.2 (17.3-18.5); into 50001 fp32 rows of 1024,
// 205 MB of zeros, 112-116 (44-45): there the sorted form would be the better one, but the entry point has no
// workspace for it.  A wave takes 16 table rows and a slab of columns, finds the rows of each
// token with a ballot over all ids and adds them in order, eight loads in flight; table rows without any
// become zeros.
template <typename D, typename W, int N>
__global__ __launch_bounds__(TE_THREADS) void tiny_sums_kernel(int n, int64_t dim, int64_t vocab, int64_t padding,
                                                               const int64_t *__restrict__ ids,
                                                               const D *__restrict__ dout, int64_t dout_stride,
                                                               float scale, W *__restrict__ dweight) {
  constexpr int K = TE_TINY / 64;
  const int lane = threadIdx.x & 63;
  const int64_t v0 = ((int64_t)blockIdx.x * (TE_THREADS / 64) + (threadIdx.x >> 6)) * 16;
  if (v0 >= vocab) return;
  const int64_t column_part = (int64_t)blockIdx.y * 64 + lane;
  const bool active = column_part * N < dim;
  const int64_t col = active ? part_column(column_part, N, dim) : 0;
  uint32_t rel[K];                                // token - v0; vocab and beyond: none
  uint64_t any = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = k * 64 + lane;
    const uint32_t token = i < n ? token_of(ids[i], vocab, padding) : (uint32_t)vocab;
    rel[k] = token < (uint32_t)vocab ? token - (uint32_t)v0 : 0xffffffffu;
    any |= __ballot(rel[k] < 16u);
  }
  for (int j = 0; j < 16 && v0 + j < vocab; ++j) {
    float acc[N];
#pragma unroll
    for (int c = 0; c < N; ++c) acc[c] = 0.f;
    bool named = false;
    if (any) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        uint64_t rows = __ballot(rel[k] == (uint32_t)j);
        named |= rows != 0;
        while (rows) {
          float x[TE_BATCH][N];
          int count = 0;
#pragma unroll
          for (int b = 0; b < TE_BATCH; ++b) {
            if (rows) {
              const int r = k * 64 + __builtin_ctzll(rows);
              rows &= rows - 1;
              load_n<N, D, true>(dout + (int64_t)r * dout_stride + col, x[b]);
              count = b + 1;
            }
          }
#pragma unroll
          for (int b = 0; b < TE_BATCH; ++b) {
            if (b >= count) break;
#pragma unroll
            for (int c = 0; c < N; ++c) acc[c] += x[b][c];
          }
        }
      }
    }
    if (named) {                                  // (0 * scale is no zero for an infinite scale)
#pragma unroll
      for (int c = 0; c < N; ++c) acc[c] *= scale;
    }
    if (active) store_n<N, W, true>(dweight + (v0 + j) * dim + col, acc);
  }
}

template <typename W>
__global__ __launch_bounds__(TE_THREADS) void zero_table_kernel(int64_t n, W *__restrict__ dweight) {
  const int64_t stride = (int64_t)gridDim.x * TE_THREADS;
  for (int64_t i = (int64_t)blockIdx.x * TE_THREADS + threadIdx.x; i < n; i += stride) dweight[i] = (W)0.f;
}

// ---------------------------------------------------------------------------------------
struct Shape {
  int64_t items, tile, tiles;
  int nblk, passes, bits;
  int64_t pairs0, pairs1, counts, part, bytes;
};
inline int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// lanes of one row: groups of 16, 32 or 64
inline int64_t lanes_of(int64_t dim, int64_t n) {
  const int64_t parts = dim < n ? dim : tv_cdiv(dim, n);
  return parts <= 16 ? 16 : parts <= 32 ? 32 : tv_cdiv(parts, 64) * 64;
}

inline Shape shape_of(int64_t rows, int64_t dim, int64_t vocab) {
  Shape s = {};
  const int64_t slots = lanes_of(dim, 8);
  int bits = 1;
  while (bits < 32 && ((int64_t)1 << bits) < vocab + 1) ++bits;
  s.passes = (int)tv_cdiv(bits, TE_MAX_BITS);
  s.bits = (int)tv_cdiv(bits, s.passes);
  // one run of ids per sort workgroup
  s.items = tv_cdiv(tv_cdiv(rows, TE_SORT_BLOCKS), TE_SORT_THREADS) * TE_SORT_THREADS;
  s.nblk = (int)tv_cdiv(rows, s.items > 0 ? s.items : 1);
  // Rows per tile: the longest that leaves 2048 waves (eight per CU), between 8 and 128.  Longer tiles leave
  // fewer sums to join, shorter ones more rows in flight: 32768 rows of 1024 bf16 into 50001 fp32 take 104, 79,
  // 72 and 74 us with tiles that leave 512, 1024, 2048 and 4096 waves, 262144 of 64 bf16 86, 69, 65 and 66;
  // 262144 of 512 bf16 in tiles of 128 take 76 us, of 256 87.
  s.tile = 8;
  while (s.tile < 128 && rows * slots / (s.tile * 2) >= 2048 * 64) s.tile *= 2;
  s.tiles = tv_cdiv(rows, s.tile);
  const bool small = rows <= TE_SMALL;
  s.pairs0 = 0;
  s.pairs1 = align256(rows * 8);
  s.counts = s.pairs1 + (s.passes > 1 && !small ? align256(rows * 8) : 0);
  s.part = s.counts + (small ? 0 : align256(s.nblk * ((int64_t)4 << s.bits)));
  s.bytes = s.part + align256(s.tiles * 2 * dim * 4);
  return s;
}

inline bool sizes_ok(int64_t rows, int64_t dim, int64_t vocab) {
  // (sorted positions and tokens fit 32 bits; a launch has less than 2^32 threads: 4 for each table row,
  // and no more than one for every 4 elements of the rows)
  return rows >= 0 && rows < INT32_MAX && dim >= 1 && dim <= (1 << 16) && vocab >= 1 && vocab <= (1 << 29) &&
         rows * lanes_of(dim, 4) < ((int64_t)1 << 33);
}

template <typename W, typename O, int N>
void launch_lookup_n(int64_t rows, int64_t dim, int64_t vocab, const void *weight, int64_t weight_stride,
                     const int64_t *ids, int64_t padding, float scale, void *out, int64_t out_stride,
                     hipStream_t stream) {
  const int parts = (int)tv_cdiv(dim, N);
  int lg = 0;
  while ((1 << lg) < parts && lg < 9) ++lg;
  const int64_t per = TE_LOOKUP_THREADS >> lg;
  // two rows per thread where that leaves two workgroups per CU (4096 x 1024 bf16 3.4 us against 3.9 with one,
  // 2048 x 1024 2.85 against 2.79)
  const bool two = tv_cdiv(rows, per) >= 1024;
  auto kernel = two ? lookup_kernel<W, O, N, 2> : lookup_kernel<W, O, N, 1>;
  const int64_t each = per * (two ? 2 : 1), most = each << 22;      // (a launch has less than 2^32 threads)
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    hipLaunchKernelGGL(kernel, dim3((unsigned)tv_cdiv(n, each)), dim3(TE_LOOKUP_THREADS), 0, stream, n, dim, vocab,
                       parts, lg, (const W *)weight, weight_stride, ids + r, padding, scale,
                       (O *)out + r * out_stride, out_stride);
  }
}
template <typename W, typename O>
void launch_lookup(int64_t rows, int64_t dim, int64_t vocab, const void *weight, int64_t weight_stride,
                   const int64_t *ids, int64_t padding, float scale, void *out, int64_t out_stride,
                   hipStream_t stream) {
  constexpr int N = 16 / sizeof(O);
  if (dim >= N)
    launch_lookup_n<W, O, N>(rows, dim, vocab, weight, weight_stride, ids, padding, scale, out, out_stride, stream);
  else
    launch_lookup_n<W, O, 1>(rows, dim, vocab, weight, weight_stride, ids, padding, scale, out, out_stride, stream);
}

void launch_sort(const Shape &s, int64_t rows, Keys keys, char *ws, hipStream_t stream) {
  uint2 *pairs[2] = {(uint2 *)(ws + s.pairs0), (uint2 *)(ws + s.pairs1)};
  if (rows <= TE_SMALL) {
    const int rounds = (int)tv_cdiv(rows, TE_SORT_THREADS);
    auto kernel = rounds <= 1 ? small_sort_kernel<1> : rounds <= 2 ? small_sort_kernel<2>
                : rounds <= 4 ? small_sort_kernel<4> : small_sort_kernel<8>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(TE_SORT_THREADS), 0, stream, (int)rows, keys, s.bits, s.passes, pairs[0]);
    return;
  }
  uint32_t *counts = (uint32_t *)(ws + s.counts);
  for (int p = 0; p < s.passes; ++p) {
    uint2 *to = pairs[(s.passes - 1 - p) & 1];    // (the last pass writes pairs[0])
    hipLaunchKernelGGL(digit_count_kernel, dim3((unsigned)s.nblk), dim3(TE_SORT_THREADS), 0, stream, rows, keys,
                       p * s.bits, s.bits, s.items, counts);
    auto scatter = s.items <= TE_SORT_THREADS ? digit_scatter_kernel<1>
                   : s.items <= 4 * TE_SORT_THREADS ? digit_scatter_kernel<4> : digit_scatter_kernel<0>;
    hipLaunchKernelGGL(scatter, dim3((unsigned)s.nblk), dim3(TE_SORT_THREADS), 0, stream, rows, keys,
                       p * s.bits, s.bits, s.items, s.nblk, counts, to);
    keys.pairs = to;
  }
}

template <typename D, typename W, int N, int G>
void launch_sums_ng(const Shape &s, int64_t rows, int64_t dim, int64_t vocab, const uint2 *sorted,
                    const void *dout, int64_t dout_stride, float scale, void *dweight, float *part,
                    hipStream_t stream) {
  const int64_t slabs = tv_cdiv(tv_cdiv(dim, N), G), units = s.tiles * slabs;
  // Rows of zeros per wave: the wider they are the fewer, so that memory is written from end to end by waves that
  // come and go.  Gradient of 32768 x 1024 into 50001 fp32 rows of 4 KB with 16, 8, 4 per wave: 85, 81, 79 us,
  // of 16384 x 1024 into 200001: 181, 168, 179; of 8192 x 4096 into 50001 bf16 rows of 8 KB: 123, 119, 111; of
  // 131072 x 256 into 100001 fp32 rows of 1 KB: 83, 85, 97.
  const int64_t bytes = dim * (int64_t)sizeof(W);
  const int zero_rows = vocab > (1 << 24) || bytes <= 1024 ? 16 : bytes <= 4096 ? 8 : 4;
  const int64_t tile_blocks = tv_cdiv(units, TE_THREADS / G);
  const int64_t zero_blocks = tv_cdiv(vocab, zero_rows * (TE_THREADS / 64));
  hipLaunchKernelGGL((tile_sums_kernel<D, W, N, G>), dim3((unsigned)(tile_blocks + zero_blocks)), dim3(TE_THREADS),
                     0, stream, rows, dim, vocab, (int)s.tile, s.tiles, slabs, tile_blocks, zero_rows, sorted,
                     (const D *)dout, dout_stride, scale, (W *)dweight, part);
  if (s.tiles > 1)
    hipLaunchKernelGGL((join_kernel<W, N, G>), dim3((unsigned)tv_cdiv(units, TE_JOIN_THREADS / G)),
                       dim3(TE_JOIN_THREADS), 0, stream, rows, dim, vocab, (int)s.tile, s.tiles, slabs, sorted,
                       scale, (W *)dweight, part);
}
template <typename D, typename W>
void launch_sums(const Shape &s, int64_t rows, int64_t dim, int64_t vocab, const uint2 *sorted,
                 const void *dout, int64_t dout_stride, float scale, void *dweight, float *part,
                 hipStream_t stream) {
  constexpr int N = 16 / sizeof(D);
  const int64_t parts = tv_cdiv(dim, N);
#define TE_NG(n, g) \
  launch_sums_ng<D, W, n, g>(s, rows, dim, vocab, sorted, dout, dout_stride, scale, dweight, part, stream)
  if (dim < N) TE_NG(1, 16);
  else if (parts <= 16) TE_NG(N, 16);
  else if (parts <= 32) TE_NG(N, 32);
  else TE_NG(N, 64);
#undef TE_NG
}

template <typename D, typename W>
void launch_tiny(int64_t rows, int64_t dim, int64_t vocab, int64_t padding, const int64_t *ids, const void *dout,
                 int64_t dout_stride, float scale, void *dweight, hipStream_t stream) {
  constexpr int N = 16 / sizeof(D);
  const dim3 grid((unsigned)tv_cdiv(vocab, 16 * (TE_THREADS / 64)),
                  (unsigned)(dim < N ? 1 : tv_cdiv(tv_cdiv(dim, N), 64)));
  auto kernel = dim < N ? tiny_sums_kernel<D, W, 1> : tiny_sums_kernel<D, W, N>;
  hipLaunchKernelGGL(kernel, grid, dim3(TE_THREADS), 0, stream, (int)rows, dim, vocab, padding, ids, (const D *)dout,
                     dout_stride, scale, (W *)dweight);
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
  return rows <= TE_TINY ? 0 : shape_of(rows, dim, num_tokens).bytes;
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
  if (rows > TE_TINY) {
    TV_REQUIRE(workspace, "tv_scaled_embedding_bwd: null workspace");
    if (workspace_bytes < s.bytes) {
      tv_set_error("tv_scaled_embedding_bwd: workspace too small");
      return TV_ERR_WORKSPACE;
    }
  }
  if (rows == 0) {
    const int64_t count = num_tokens * dim;
    int64_t blocks = tv_cdiv(count, TE_THREADS * 8);
    if (blocks > 16384) blocks = 16384;
    if (weight_dtype == TV_DTYPE_F32)
      hipLaunchKernelGGL(zero_table_kernel<float>, dim3((unsigned)blocks), dim3(TE_THREADS), 0, st, count,
                         (float *)dweight);
    else
      hipLaunchKernelGGL(zero_table_kernel<_Float16>, dim3((unsigned)blocks), dim3(TE_THREADS), 0, st, count,
                         (_Float16 *)dweight);
    TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
    return TV_OK;
  }
#define TE_GO_ALL                                                                           \
  if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_F32) TE_GO(float, float);       \
  else if (weight_dtype == TV_DTYPE_F32 && out_dtype == TV_DTYPE_BF16) TE_GO(__bf16, float); \
  else if (weight_dtype == TV_DTYPE_F32) TE_GO(_Float16, float);                            \
  else if (weight_dtype == TV_DTYPE_BF16) TE_GO(__bf16, __bf16);                            \
  else TE_GO(_Float16, _Float16)
  if (rows <= TE_TINY) {
#define TE_GO(D, W) \
  launch_tiny<D, W>(rows, dim, num_tokens, padding_id, ids, dout, dout_stride, scale, dweight, st)
    TE_GO_ALL;
#undef TE_GO
    TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
    return TV_OK;
  }
  char *ws = (char *)workspace;
  launch_sort(s, rows, Keys{ids, nullptr, num_tokens, padding_id}, ws, st);
  TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
  const uint2 *sorted = (const uint2 *)(ws + s.pairs0);
  float *part = (float *)(ws + s.part);
#define TE_GO(D, W) launch_sums<D, W>(s, rows, dim, num_tokens, sorted, dout, dout_stride, scale, dweight, part, st)
  TE_GO_ALL;
#undef TE_GO
#undef TE_GO_ALL
  TV_LAUNCH_CHECK("tv_scaled_embedding_bwd");
  return TV_OK;
}
