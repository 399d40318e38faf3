// r3_ortho.hip -- orthogonalising the updates of weight matrices by Newton-Schulz products, for a ragged list of matrices at
// once, alone or inside the optimiser's step (momentum before it, the weights' update behind it).
//
// For a matrix G (n x m, n <= m; a taller one is taken transposed):
//   X = G / (|G|_F + eps);   per step:  A = X X^t,  B = b A + c A A,  X <- a X + B X
// Each singular value s goes to a s + b s^3 + c s^5 while the singular vectors stay.  With the usual coefficients a small one
// grows by a = 3.44 a step, 485 in five, and so does every rounding of X: iterates rounded to 16 bits leave an error of
// 2-3 % in the result where the spectrum is a few directions over noise (fp16; 20 % in bf16).  So an iterate is held as
// TWO fp16 numbers, hi + lo, 22 bits and lo's sign, and a product is three matrix products on the matrix cores,
// hi hi + (hi lo + lo hi), summed in fp32 in two accumulators.
//
// Steps are taken in groups of two (the first of three where their number is odd) that touch X only twice; short lists and
// matrices of fewer than 256 rows take them one by one (NARROW below).  Everything inside a group is a polynomial of its first A, n x n and symmetric, written without
// cancellation: with the square completed, t = -b / 2c and q = a - c t^2, a step multiplies X by
//   F = a I + b A + c A A = q I + c (A - t I)^2,
// which for the usual coefficients is 0.64 I and a positive matrix (the three terms cancel six to one where singular values
// are near 1).  The next A is F (F A), and the group's steps together are X <- R X with R the product of the F.
// For m = 9 n (a 3 x 3 convolution of equal width) that halves the operations and reads X twice instead of five times; a
// square matrix needs as many operations as before.  Longer groups at the end lose digits (2 + 3 twice the error of 3 + 2).
//
// The symmetric matrices are mostly diagonal -- A is near I where it has converged, and far from it F is near a I -- and
// the diagonal would decide where the matrix cores round.  It is kept apart, in fp32, and products take it apart:
//   (G H)_ij = g_i H_ij + h_j G_ij + sum_k G_ik H_kj  with G and H without their diagonals,  (G H)_ii = g_i h_i + the sum.
//
// Stored values carry a power of two so that fp16 neither overflows -- spectral norms bound the entries, and the host checks
// them for the given coefficients -- nor loses lo's bits: 2^12 for X, A, F, F A (norms below 15), 2^9 for R and what is made of it
// (below 120).
//
// The matrix instructions want both operands with the summed index contiguous.  The symmetric matrices and X X^t have it;
// for R X, X is turned on its way out of shared memory (tiles of 128), or X^t is kept beside it (tiles of 64, which come
// straight from memory).  Of a symmetric result the tiles on and above the diagonal are computed, and written twice.
//
// What bounds it, with the usual five steps (kernels' time of a call; the matrix cores reach 1.1 PFLOP/s of fp16, a copy
// 4.7 TB/s): 4096 x 4096, 4.6 ms: the matrix cores, 3.75 ms of products at that rate.  2048 x 2048, 0.95 ms: the same, with
// fewer tiles than would keep them busy (0.47).  The 73 matrices of a detector, 41.9 M weights, 1.27 ms: a third the memory
// (norms 87 us, X 105, the last launch 213), the rest loads on their way between matrix instructions.  A head's ten,
// 0.25 ms, and smaller lists: some twenty-five launches that wait for each other, 5 us at least each.
#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

#include "../r3_kernels.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float SCALE = 4096.f;  // what stored values are multiplied by
constexpr float R_SCALE = 512.f; // ... of R
constexpr int PAD = 128;         // rows and columns of X are multiples of it
constexpr int WANT = 512;        // workgroups that fill the card
constexpr unsigned CARD = 256;   // its compute units

struct Mat {  // one matrix, as the device's table holds it
  const void* src;   // the matrix / the gradient
  void* dst;         // the result / the weights
  float* buf;        // the momentum (update only)
  int rows, cols;    // as the caller has it
  float rate;        // weights <- decay * weights - rate * result
  unsigned splits;   // parts of the sum of X X^t
  unsigned gram0, tri0, rect0, fill0, norm0;  // first entries in the lists, see Lists
  size_t part0;      // floats before this matrix's partial tiles
  size_t at;         // halves before this matrix's arrays
};
__host__ __device__ inline int up(int v, int to) { return (v + to - 1) / to * to; }
enum { SQ_A, SQ_FA, SQ_F, SQ_R = SQ_F + 2, SQ = SQ_R + 2 };  // (two of F, two of R)
struct Dim {  // padded with zeros, which stay zeros
  int n, m, np, mp;
  __host__ __device__ Dim(int rows, int cols) {
    n = rows < cols ? rows : cols;
    m = rows < cols ? cols : rows;
    np = up(n, PAD), mp = up(m, PAD);
  }
  __host__ __device__ size_t x() const { return (size_t)np * mp; }
  __host__ __device__ size_t a() const { return (size_t)np * np; }
  // per matrix: X twice (one read and one written in a pass), or X and X^t twice; SQ n x n arrays, each hi then lo; SQ
  // diagonals in fp32
  __host__ __device__ size_t halves(int rect_ts) const { return 2 * ((rect_ts == 64 ? 3 : 2) * x() + SQ * a() + (size_t)SQ * np); }
  __host__ __device__ unsigned tri(int ts) const { return (unsigned)(np / ts) * (np / ts + 1) / 2; }
  __host__ __device__ unsigned rect(int ts) const { return (unsigned)(np / ts) * (mp / ts); }
  __host__ __device__ unsigned norms(int chunk) const { return (unsigned)(((size_t)n * m + chunk - 1) / chunk); }
};
struct Tile {  // one workgroup's work, with all that it needs of its matrix to begin
  size_t at;    // Mat::at
  size_t part;  // X X^t in parts: where this one goes
  int np, mp;
  unsigned short i, j, split, splits;
  unsigned short ts;  // 128 or 64 rows and columns (0: none), in units of which i and j are; fill: the chain's rect_ts
  unsigned mat;
};
struct Area {  // where a matrix's arrays are
  _Float16 *x, *next, *sq;  // X (or X^t) that a pass reads, and writes; sq: SQ
  _Float16 *xt, *next_t;
  float* diag;
  size_t na;  // one of sq's (hi and lo)
  __device__ Area(_Float16* base, const Tile& t, int rect_ts, int from) {
    const size_t nx = 2 * (size_t)t.np * t.mp;
    na = 2 * (size_t)t.np * t.np;
    x = next = base + t.at;
    sq = x + (rect_ts == 64 ? 3 : 2) * nx;
    diag = reinterpret_cast<float*>(sq + SQ * na);
    if (rect_ts == 64) xt = x + (from ? 2 : 1) * nx, next_t = x + (from ? 1 : 2) * nx;
    else xt = next_t = nullptr, x += from ? nx : 0, next += from ? 0 : nx;
  }
};
struct Chain {  // lists of a chain of launches, one entry a workgroup
  Tile* gram;  // X X^t: triangle tiles times parts of the sum
  Tile* tri;   // triangle tiles of the other n x n products
  Tile* rect;  // tiles of X
  unsigned n_gram, n_tri, n_rect;
  unsigned whole_gram, whole_tri;  // tiles that are not quartered
  int gram_ts, tri_ts, rect_ts;
  unsigned gram0, tri0, rect0;     // of its first matrix, see Mat
};
struct Lists {
  Mat* table;       // of one chain's matrices behind the other's
  Tile* fill;       // 64 x 64 pieces of X
  uint2* norm_map;  // (matrix, chunk)
  unsigned n_fill, n_norm;
  unsigned second;  // the second chain's first matrix
  int chunk;        // elements a workgroup of the norm's pass takes
  Chain c[2];
};

// ------------------------------------------------------------------------------------------------ the lists
constexpr int BATCH = 40;
struct Batch {
  Mat m[BATCH];
  int count;
  Mat end;  // behind the last: the lists' ends
};
static_assert(sizeof(Batch) <= 3800, "a kernel's arguments hold 4 KB");

__device__ __forceinline__ unsigned find(const Batch& b, unsigned Mat::* first, unsigned e) {
  int lo = 0, hi = b.count - 1;  // the last matrix that begins at or before e
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (b.m[mid].*first <= e) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// The tile-th of the tiles on and above the diagonal, `wide` by `wide` of them: in squares of SIDE, row by row of squares,
// each row by row.
constexpr unsigned SIDE = 8;
__device__ __forceinline__ void triangle(Tile& w, unsigned tile, unsigned wide) {
  unsigned i = 0, j = 0;
  for (;;) {  // the square whose first tile is (i, j)
    const unsigned high = wide - i < SIDE ? wide - i : SIDE, across = wide - j < SIDE ? wide - j : SIDE;
    const unsigned many = i == j ? high * (high + 1) / 2 : high * across;
    if (tile < many) {
      if (i == j) {
        unsigned r = 0;
        while (tile >= high - r) tile -= high - r, ++r;  // (row r has high - r tiles)
        w.i = i + r, w.j = j + r + tile;
      } else {
        w.i = i + tile / across, w.j = j + tile % across;
      }
      return;
    }
    tile -= many;
    j += SIDE;
    if (j >= wide) i += SIDE, j = i;
  }
}
// Workgroups go to the eight XCDs in turn, and each has an L2 of its own.  The u-th of n pieces of work is taken by that
// workgroup which makes CHUNK neighbours share one: the tiles of a matrix read the same rows (a head's X X^t: 12.5 us, 16.9
// in the order as it comes; n x n products of a ragged list: 14.1, 17.2).  8, 32 and 64 of them do as well there, but 64 puts
// a long list's largest matrices on one XCD.
constexpr unsigned XCDS = 8, CHUNK = 16;
__device__ __forceinline__ unsigned entry(unsigned u, unsigned n) {
  const unsigned first = u / (XCDS * CHUNK) * (XCDS * CHUNK), v = u - first;
  const unsigned here = n - first < XCDS * CHUNK ? n - first : XCDS * CHUNK;  // (fewer at the end: as even as possible)
  const unsigned q = here / XCDS, longer = here % XCDS * (q + 1);
  const unsigned x = v < longer ? v / (q + 1) : here % XCDS + (v - longer) / q;
  const unsigned c = v < longer ? v % (q + 1) : (v - longer) % q;
  return first + c * XCDS + x;
}
// the table's and the lists' entries of `b`'s matrices: a thread an entry, list behind list
__global__ void ortho_lists_kernel(Lists l, Batch b, unsigned first) {
  unsigned e = blockIdx.x * blockDim.x + threadIdx.x;
  if (e < (unsigned)b.count) l.table[first + e] = b.m[e];
  const auto within = [&](unsigned Mat::* member) {  // of this list: the entry, and the matrix in front of which it begins
    const unsigned from = b.m[0].*member, many = b.end.*member - from;
    if (e < many) {
      e += from;
      return true;
    }
    e -= many;
    return false;
  };
  const auto begin = [&](unsigned k) {
    const Mat& t = b.m[k];
    const Dim d(t.rows, t.cols);
    return Tile{t.at, 0, d.np, d.mp, 0, 0, 0, (unsigned short)t.splits, 0, first + k};
  };
  // the u-th tile of a triangle list, of n as they are and of 64 x 64 quarters behind those
  const auto put = [&](Tile* list, Tile w, unsigned u, unsigned n, int ts) {
    w.ts = ts;
    if (u < n) {
      list[entry(u, n)] = w;
      return;
    }
    for (unsigned q = 0; q < 4; ++q) {
      Tile v = w;
      v.i = 2 * w.i + q / 2, v.j = 2 * w.j + q % 2;
      v.ts = v.i <= v.j ? 64 : 0;
      list[n + 4 * (u - n) + q] = v;
    }
  };
  const auto chain = [&](unsigned k) -> const Chain& { return l.c[first + k >= l.second]; };
  if (within(&Mat::gram0)) {
    const unsigned k = find(b, &Mat::gram0, e), local = e - b.m[k].gram0;
    const Chain& c = chain(k);
    Tile w = begin(k);
    const unsigned high = w.np / c.gram_ts, tiles = high * (high + 1) / 2, tile = local % tiles;
    triangle(w, tile, high);
    w.split = local / tiles;
    w.part = b.m[k].part0 + ((size_t)tile * w.splits + w.split) * (c.gram_ts * c.gram_ts);
    put(c.gram, w, e - c.gram0, c.whole_gram, c.gram_ts);
  } else if (within(&Mat::tri0)) {
    const unsigned k = find(b, &Mat::tri0, e);
    const Chain& c = chain(k);
    Tile w = begin(k);
    triangle(w, e - b.m[k].tri0, w.np / c.tri_ts);
    put(c.tri, w, e - c.tri0, c.whole_tri, c.tri_ts);
  } else if (within(&Mat::rect0)) {
    const unsigned k = find(b, &Mat::rect0, e), local = e - b.m[k].rect0;
    const Chain& c = chain(k);
    Tile w = begin(k);
    const unsigned high = w.np / c.rect_ts;
    w.i = local % high, w.j = local / high;
    c.rect[entry(e - c.rect0, c.n_rect)] = w;
  } else if (within(&Mat::fill0)) {
    const unsigned k = find(b, &Mat::fill0, e), local = e - b.m[k].fill0;
    Tile w = begin(k);
    const unsigned wide = w.mp / 64;
    w.i = local / wide, w.j = local % wide;
    w.ts = chain(k).rect_ts;
    l.fill[e] = w;
  } else if (within(&Mat::norm0)) {
    const unsigned k = find(b, &Mat::norm0, e);
    l.norm_map[e] = make_uint2(first + k, e - b.m[k].norm0);
  }
}

// ------------------------------------------------------------------------------------------------ momentum, norm, X
// N elements as one, from an address that is aligned to one of them: global accesses need no more.
template <typename T, int N>
struct Few {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Few<T, N> load_few(const T* at) {
  Few<T, N> x;
  __builtin_memcpy(&x, at, sizeof(x));
  return x;
}
template <typename T, int N>
__device__ __forceinline__ void store_few(T* at, const Few<T, N>& x) {
  __builtin_memcpy(at, &x, sizeof(x));
}
// What is orthogonalised, N elements from i on: the matrix, or the gradient with the momentum (new: after its update, which
// this is).
struct Momentum {
  int update, nesterov;
  float mu;
};
template <typename T, int N, bool NEW>
__device__ __forceinline__ void direction(float (&v)[N], const Mat& t, size_t i, const Momentum& m) {
  const Few<T, N> g = load_few<T, N>(static_cast<const T*>(t.src) + i);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = (float)g.v[k];
  if (!m.update) return;
  Few<float, N> b = load_few<float, N>(t.buf + i);
  if constexpr (NEW) {
#pragma unroll
    for (int k = 0; k < N; ++k) b.v[k] = fmaf(m.mu, b.v[k], v[k]);
    store_few(t.buf + i, b);
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = m.nesterov ? fmaf(m.mu, b.v[k], v[k]) : b.v[k];
}
template <int THREADS = 256>
__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; w += 4) v += (sh[w] + sh[w + 1]) + (sh[w + 2] + sh[w + 3]);
  return v;
}
// momentum <- mu momentum + gradient, and the squares of the direction summed in 64 bits (no scaling of the matrix is needed
// against overflow, and the order of the sums is fixed)
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(Lists l, double* __restrict__ norms, Momentum m) {
  __shared__ double sh[4];
  const uint2 w = l.norm_map[blockIdx.x];
  const Mat t = l.table[w.x];
  const size_t all = (size_t)t.rows * t.cols, from = (size_t)w.y * l.chunk;
  const int many = (int)(from + l.chunk < all ? l.chunk : all - from);
  double s = 0;
#pragma unroll 4
  for (int q = threadIdx.x; q < many / 4; q += 256) {
    float v[4];
    direction<T, 4, true>(v, t, from + 4 * q, m);
#pragma unroll
    for (int k = 0; k < 4; ++k) s = fma((double)v[k], (double)v[k], s);
  }
  for (int i = many / 4 * 4 + threadIdx.x; i < many; i += 256) {
    float v[1];
    direction<T, 1, true>(v, t, from + i, m);
    s = fma((double)v[0], (double)v[0], s);
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) norms[blockIdx.x] = s;
}
// A TS x TS tile at (i0, j0) in the caller's order, elements N at a time along the caller's rows (a constant: 4, or 1 where a
// row has fewer): x = load(N, place, how many are inside), then f(N, place, how many, row and column in the tile of the
// first, TALL, x).  TALL: the tile is of the transpose.  BATCH loads, then as many f.  PARTS: N may be cut by the row's end.
template <int N, bool PARTS>
struct Many {
  static constexpr bool parts = PARTS;
  __device__ constexpr int operator()() const { return N; }
};
template <int TS, int BATCH, int N, bool PARTS, typename Load, typename F>
__device__ __forceinline__ void callers_by(const Mat& t, int i0, int j0, const Load& load, const F& f) {
  const Many<N, PARTS> n;
  const bool tall = t.rows > t.cols;
  const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;
  for (int from = 0; from < TS * TS / N; from += 256 * BATCH) {
    decltype(load(n, 0, 0)) x[BATCH];
    const auto each = [&](int b, const auto& g) {
      const int q = from + b * 256 + threadIdx.x, r = q / (TS / N), c = q % (TS / N) * N, left = t.cols - (c0 + c);
      g((size_t)(r0 + r) * t.cols + c0 + c, r0 + r < t.rows && left > 0 ? (left < N ? left : N) : 0, tall ? c : r, tall ? r : c);
    };
#pragma unroll
    for (int b = 0; b < BATCH; ++b) each(b, [&](size_t at, int many, int, int) { x[b] = load(n, at, many); });
#pragma unroll
    for (int b = 0; b < BATCH; ++b) each(b, [&](size_t at, int many, int r, int c) { f(n, at, many, r, c, tall, x[b]); });
  }
}
template <int TS, int BATCH, typename Load, typename F>
__device__ __forceinline__ void callers(const Mat& t, int i0, int j0, const Load& load, const F& f) {
  constexpr int FOURS = TS * TS / 4 / 256;
  constexpr int EACH = BATCH < FOURS ? BATCH : FOURS;
  if (t.cols % 4 == 0) callers_by<TS, EACH, 4, false>(t, i0, j0, load, f);
  else if (t.cols >= 4) callers_by<TS, EACH, 4, true>(t, i0, j0, load, f);
  else callers_by<TS, BATCH, 1, false>(t, i0, j0, load, f);
}
// What `many` elements of N at `at` are read from, whole and inside the row: so many places before as are missing (0:
// anywhere, from the array's beginning); then they are the last of the N read.
template <typename N>
__device__ __forceinline__ size_t whole(const N& n, size_t at, int many) {
  return many ? at - (N::parts ? n() - many : 0) : 0;
}
template <typename N, typename T, int COUNT>
__device__ __forceinline__ void to_front(const N&, T (&v)[COUNT], int many) {
  if constexpr (N::parts) {
    const T a = v[1], b = v[2], c = v[3];
    v[0] = many == 3 ? a : many == 2 ? b : many == 1 ? c : v[0];
    v[1] = many == 3 ? b : many == 2 ? c : a;
    v[2] = many == 3 ? c : b;
  }
}

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}
// Arrays are kept in blocks of 64 rows by 32 columns, row by row of blocks: 4 KB of hi, 4 KB of lo.  Inside, in the order of
// the matrix instruction's operands: 16 columns, 32 rows, 8 columns, row, column, so that a wavefront's operand is 1 KB in
// one piece.  What a stage of a product reads is then whole blocks, one behind the other.  (Plain rows are read 64 bytes at
// a time, half a cache line, and at a power of two apart: 7.0 ms for 4096 x 4096 against 6.2.)
constexpr int LO = 64 * 32, BLOCK = 2 * LO;
__device__ __forceinline__ size_t place(int r, int c, int ld) {
  return ((size_t)(r / 64) * (ld / 32) + c / 32) * BLOCK + c % 32 / 16 * 1024 + r % 64 / 32 * 512 + c % 16 / 8 * 256 + r % 32 * 8 +
         c % 8;
}
__device__ __forceinline__ void store8(_Float16* at, const float (&v)[8]) {
  half8 h, l;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    _Float16 hh, ll;
    split16(v[k], hh, ll);
    h[k] = hh, l[k] = ll;
  }
  *reinterpret_cast<half8*>(at) = h;
  *reinterpret_cast<half8*>(at + LO) = l;
}
struct Both {
  half8 h, l;
  __device__ __forceinline__ float operator[](int k) const { return (float)h[k] + (float)l[k]; }
};
__device__ __forceinline__ Both load8(const _Float16* at) {
  return Both{*reinterpret_cast<const half8*>(at), *reinterpret_cast<const half8*>(at + LO)};
}
// ROWS x COLS of fp32 in shared memory, rows of LD: f(row, column, eight values), which may change them; then `f`'s values
// are in shared memory too.  PARTS > 1: the values are the sum of so many such arrays.  (Neighbouring threads have
// neighbouring rows: the arrays' order, and LD is odd.)
template <int LD, int PARTS, int STRIDE, typename F>
__device__ __forceinline__ void eight(float* E, int r, int c, const F& f) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = E[r * LD + c + k];
#pragma unroll
  for (int s = 1; s < PARTS; ++s)
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += E[s * STRIDE + r * LD + c + k];
  f(r, c, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) E[r * LD + c + k] = v[k];
}
template <int ROWS, int COLS, int LD, int PARTS, int THREADS = 256, typename F>
__device__ __forceinline__ void rows8(float* E, const F& f) {
#pragma unroll 2
  for (int q = threadIdx.x; q < ROWS * COLS / 8; q += THREADS) eight<LD, PARTS, ROWS * LD>(E, q % ROWS, q / ROWS * 8, f);
}
// The same for a product's tile, where f takes what `load`(row, column) gives too: loaded for several rows at a time, the
// first of them before the product's sums are in shared memory.  (What f stores could be what the next row loads, for all
// that the compiler knows: it would wait for each.)
template <typename C, typename Load>
struct Rows {
  static constexpr int N = C::TS * C::TS / 8 / C::THREADS, BATCH = N < 4 ? N : 4;
  const Load& load;
  decltype(load(0, 0)) d[BATCH];
  __device__ __forceinline__ void fetch(int from) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int q = (from + b) * C::THREADS + threadIdx.x;
      d[b] = load(q % C::TS, q / C::TS * 8);
    }
  }
  template <typename F>
  __device__ __forceinline__ void run(float* E, const F& f) {
    for (int from = 0; from < N; from += BATCH) {
      if (from) fetch(from);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int q = (from + b) * C::THREADS + threadIdx.x;
        eight<C::LD, C::PARTS, C::TS * C::LD>(E, q % C::TS, q / C::TS * 8,
                                              [&](int r, int c, float (&v)[8]) { f(r, c, v, d[b]); });
      }
    }
  }
};
// The transpose of ROWS x COLS in shared memory -> an array of `ld` columns, at (r0, c0).
template <int ROWS, int COLS, int LD, int THREADS = 256>
__device__ __forceinline__ void store_turned(const float* E, _Float16* p, int ld, int r0, int c0) {
#pragma unroll 2
  for (int q = threadIdx.x; q < ROWS * COLS / 8; q += THREADS) {
    const int r = q % COLS, c = q / COLS * 8;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = E[(c + k) * LD + r];
    store8(p + place(r0 + r, c0 + c, ld), v);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ortho_start_kernel(Lists l, const double* __restrict__ norms,
                                                          _Float16* __restrict__ base, Momentum m, double eps) {
  __shared__ double sh[4];
  __shared__ float E[64 * 65];
  const Tile w = l.fill[blockIdx.x];
  const Mat t = l.table[w.mat];
  const Area o(base, w, w.ts, 0);
  double s = 0;
  const unsigned chunks = Dim(t.rows, t.cols).norms(l.chunk);
  for (unsigned i = threadIdx.x; i < chunks; i += 256) s += norms[t.norm0 + i];
  s = block_sum(s, sh);
  const double inv = (double)SCALE / (sqrt(s) + eps);
  const int i0 = w.i * 64, j0 = w.j * 64;
  callers<64, 4>(
      t, i0, j0,
      [&](auto N, size_t at, int many) {  // (inside or not, so that several are on their way)
        Few<float, N()> x;
        direction<T, N(), false>(x.v, t, whole(N, at, many), m);
        to_front(N, x.v, many);
        return x;
      },
      [&](auto N, size_t, int many, int r, int c, bool tall, const auto& x) {
#pragma unroll
        for (int k = 0; k < N(); ++k)
          E[(tall ? r + k : r) * 65 + (tall ? c : c + k)] = (decltype(N)::parts ? k < many : many != 0) ? (float)((double)x.v[k] * inv) : 0.f;
      });
  __syncthreads();
  rows8<64, 64, 65, 1>(E, [&](int r, int c, float (&v)[8]) { store8(o.x + place(i0 + r, j0 + c, w.mp), v); });
  if (o.xt) store_turned<64, 64, 65>(E, o.xt, w.np, j0, i0);
}

// ------------------------------------------------------------------------------------------------ the products
// One TS x TS tile of P Q^t by 4 wavefronts: P, Q arrays of ldp / ldq columns, of which [k0, k1) are summed, a multiple of 128;
// the tile's first rows given.  Three matrix instructions for two operands of hi and lo, in two accumulators.
typedef float16v Acc[2][2];
__device__ __forceinline__ void clear(Acc& a) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) a[i][j] = float16v{};
}
struct Piece {  // 64 rows of P and of Q, 16 of the summed index
  half8 ph[2], pl[2], qh[2], ql[2];
};
__device__ __forceinline__ void multiply(Acc& hh, Acc& hl, const Piece& f) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) hl[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[i], f.ql[j], hl[i][j], 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) hh[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ph[i], f.qh[j], hh[i][j], 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) hl[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.pl[i], f.qh[j], hl[i][j], 0, 0, 0);
}
// 64 x 64 of the sum, into shared memory with rows of LD, times f.  Lane l of the matrix instruction holds column l % 32 and
// rows 8 (r / 4) + 4 (l / 32) + r % 4.
template <int LD>
__device__ __forceinline__ void spill(const Acc& hh, const Acc& hl, float* E, float f) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        E[(32 * i + 8 * (r / 4) + 4 * (lane >> 5) + r % 4) * LD + 32 * j + (lane & 31)] = (hh[i][j][r] + hl[i][j][r]) * f;
}

// A tile of 128: a quarter a wavefront.  A stage is 32 of the summed index, whole blocks; it comes through registers into
// shared memory, two stages in turn, two workgroups a compute unit.  The next stage's loads, the writes of the one before
// it and the reads of the second piece lie between the matrix instructions, in an order that the scheduler is told:
// left alone it reads an operand where it is needed and waits (R X of 4096 x 4096: 395 us, 387 with it; of 2048 x 2048: 74, 61).
// Nothing is conditional -- the last stage is loaded again where there is no next -- or the compiler could not count the
// loads in flight and would wait for all of them.  (Loads straight into shared memory do not overlap: before any of it is
// read, the compiler waits for every such load in flight.)  The 16-byte pieces of a row change places
// with its number: sixteen rows that are read together lie in different banks, and so do eight that are written together
// in the 32 banks that a write reaches at a time (no conflicts; a third of the cycles with the order that only the reads
// need, X X^t of 4096 x 4096: 261 us, 255 so).
struct Stage {
  half8 v[4][512];
};
struct Core128 {
  static constexpr int TS = 128, LD = 129, PARTS = 1, THREADS = 256;
  static constexpr int MFMA = 8, VMEM_READ = 0x20, DS_READ = 0x100, DS_WRITE = 0x200;  // kinds of instructions
  union Shared {
    Stage st[2];
    float E[TS * LD];
  };
  struct Source {  // the first stage's blocks
    const _Float16 *p[2], *q[2];
    size_t down;  // TURNED: 64 rows further in Q
  };
  static __device__ __forceinline__ int spot(int r, int c) { return r * 4 + (c ^ (r / 4 % 2 + (r / 2 ^ r / 8) % 2 * 2)); }
  // TURNED: Q's rows are the summed index.  (R X of 4096 x 4096: 390 us, of 2048 x 2048 70; 388 and 66 from an X^t, which
  // has to be written and read beside X: R X of the detector's matrices 184 + 215 us so and their first X 129, against
  // 162 + 213 and 99.)  32 of them lie in shared memory as they come, the 16-byte piece c of row k at
  // this place, and are turned by the reads of it: of sixteen lanes, four each name sixteen columns of a row, and each
  // receives four rows of a column.  Both ways go over all banks.
  static __device__ __forceinline__ int turned_spot(int k, int c) {
    return k * 16 + (c / 4 ^ k % 4) * 4 + (c % 4 ^ (k / 4 % 2 + k / 2 % 2 * 2));
  }
  template <bool TURNED>
  static __device__ __forceinline__ void fetch(half8 (&to)[8], const Source& s, int stage) {
    const size_t k = (size_t)stage * BLOCK + threadIdx.x * 8;
    const size_t kq = TURNED ? (size_t)(stage / 2) * s.down + stage % 2 * 512 + threadIdx.x % 64 * 8 : k;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      to[4 * t] = *reinterpret_cast<const half8*>(s.p[t] + k);
      to[4 * t + 1] = *reinterpret_cast<const half8*>(s.p[t] + k + LO);
      to[4 * t + 2] = *reinterpret_cast<const half8*>(s.q[t] + kq);
      to[4 * t + 3] = *reinterpret_cast<const half8*>(s.q[t] + kq + LO);
    }
  }
  template <bool TURNED>
  static __device__ __forceinline__ void put(Stage& s, const half8 (&from)[8]) {
    const int t4 = threadIdx.x, r = t4 / 64 % 2 * 32 + t4 % 32, c = t4 / 128 * 2 + t4 / 32 % 2;  // (the block's order)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int ps = spot(t * 64 + r, c), qs = TURNED ? turned_spot(t4 % 32, t * 8 + t4 / 32) : ps;
      s.v[0][ps] = from[4 * t], s.v[1][ps] = from[4 * t + 1], s.v[2][qs] = from[4 * t + 2], s.v[3][qs] = from[4 * t + 3];
    }
  }
  static __device__ __forceinline__ half4 turn(const half8* at, int half) {
    typedef __attribute__((address_space(3))) decltype(__builtin_amdgcn_ds_read_tr16_b64_v4f16(nullptr)) Turned;
    const auto v = __builtin_amdgcn_ds_read_tr16_b64_v4f16((Turned*)(reinterpret_cast<const half4*>(at) + half));
    return __builtin_bit_cast(half4, v);
  }
  template <bool TURNED>
  static __device__ __forceinline__ void read(Piece& f, const Stage& s, int kk) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int pr = (wave >> 1) * 64 + (lane & 31), qr = (wave & 1) * 64 + (lane & 31), kc = lane >> 5;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ps = spot(pr + 32 * i, kk * 2 + kc);
      f.ph[i] = s.v[0][ps], f.pl[i] = s.v[1][ps];
      if constexpr (TURNED) {
        const int c = (wave & 1) * 8 + 4 * i + lane / 16 % 2 * 2 + lane % 4 / 2, k = kk * 16 + kc * 8 + lane % 16 / 4;
        const int one = turned_spot(k, c), two = turned_spot(k + 4, c);
        f.qh[i] = __builtin_shufflevector(turn(&s.v[2][one], lane & 1), turn(&s.v[2][two], lane & 1), 0, 1, 2, 3, 4, 5, 6, 7);
        f.ql[i] = __builtin_shufflevector(turn(&s.v[3][one], lane & 1), turn(&s.v[3][two], lane & 1), 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        const int qs = spot(qr + 32 * i, kk * 2 + kc);
        f.qh[i] = s.v[2][qs], f.ql[i] = s.v[3][qs];
      }
    }
  }
  // the tile times f in shared memory; TURNED: of P Q; `before` is called when the sums are done
  template <bool TURNED = false, typename Before>
  static __device__ __forceinline__ void run(Shared& sh, const _Float16* p, int prow, int ldp, const _Float16* q, int qrow,
                                             int ldq, int k0, int k1, float f, const Before& before) {
    Source src;
    src.down = (size_t)(ldq / 32) * BLOCK;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      src.p[t] = p + place(prow + 64 * t, k0, ldp);
      src.q[t] = q + (TURNED ? place(k0, qrow + 64 * t + threadIdx.x / 64 * 16, ldq) : place(qrow + 64 * t, k0, ldq));
    }
    const int stages = (k1 - k0) / 32, end = stages - 1;
    half8 next[8];
    Piece one, two;
    Acc hh, hl;
    fetch<TURNED>(next, src, 0);
    clear(hh), clear(hl);
    put<TURNED>(sh.st[0], next);
    fetch<TURNED>(next, src, 1);
    __syncthreads();
    Stage *now = sh.st, *then = sh.st + 1;
    for (int s = 0; s < stages; ++s) {
      read<TURNED>(one, *now, 0);
      read<TURNED>(two, *now, 1);
      multiply(hh, hl, one);
      put<TURNED>(*then, next);  // (that stage was left before the last barrier)
      fetch<TURNED>(next, src, s + 2 < end ? s + 2 : end);
      multiply(hh, hl, two);
      constexpr int READS = TURNED ? 12 : 8, LOADS = TURNED ? 2 : 1;  // (24 matrix instructions)
#pragma unroll
      for (int k = 0; k < READS; ++k) __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
#pragma unroll
      for (int k = 0; k < READS; ++k) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(DS_READ, 1, 0);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(DS_WRITE, 1, 0);
      }
#pragma unroll
      for (int k = 0; k < 8 / LOADS; ++k) {
        __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
        __builtin_amdgcn_sched_group_barrier(VMEM_READ, LOADS, 0);
      }
      __syncthreads();  // (behind the last stage: the stages' memory is the epilogue's too)
      Stage* was = now;
      now = then, then = was;
    }
    before();
    const int wave = threadIdx.x >> 6;
    spill<LD>(hh, hl, sh.E + (wave >> 1) * 64 * LD + (wave & 1) * 64, f);
    __syncthreads();
  }
};

// A tile of 64, for where those of 128 are too few: the whole tile a wavefront, the summed index in turn, 16 of it at a time.
// Operands come from memory straight into registers, each by one wavefront only, so shared memory has nothing to save and
// nobody waits at a barrier before the end; there the wavefronts' sums are added.  Two pieces are on their way (three, and
// loads of the last one again where there is no next: 9 more where a wavefront has four; 64 x 64 of 256: 9.2 us, 8.4 so).
template <int WAVES>
struct Core64 {
  static constexpr int TS = 64, LD = 65, PARTS = WAVES, THREADS = 64 * WAVES, AHEAD = 2;
  union Shared {
    float E[PARTS * TS * LD];
  };
  static __device__ __forceinline__ void fetch(Piece& f, const _Float16* p, const _Float16* q, int unit) {
    const size_t k = (size_t)(unit / 2) * BLOCK + unit % 2 * 1024 + (threadIdx.x & 63) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f.ph[i] = *reinterpret_cast<const half8*>(p + k + i * 512);
      f.pl[i] = *reinterpret_cast<const half8*>(p + k + i * 512 + LO);
      f.qh[i] = *reinterpret_cast<const half8*>(q + k + i * 512);
      f.ql[i] = *reinterpret_cast<const half8*>(q + k + i * 512 + LO);
    }
  }
  template <typename Before>
  static __device__ __forceinline__ void run(Shared& sh, const _Float16* p, int prow, int ldp, const _Float16* q, int qrow,
                                             int ldq, int k0, int k1, float f, const Before& before) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    p += place(prow, k0, ldp), q += place(qrow, k0, ldq);
    const int units = (k1 - k0) / (16 * WAVES), end = units - 1;  // of this wavefront
    Piece piece[AHEAD];
    Acc hh, hl;
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) fetch(piece[d], p, q, (d < end ? d : end) * WAVES + wave);
    clear(hh), clear(hl);
    int s = 0;
    for (; s + AHEAD < units; s += AHEAD) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        multiply(hh, hl, piece[u]);
        fetch(piece[u], p, q, (s + u + AHEAD < end ? s + u + AHEAD : end) * WAVES + wave);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (s + u < units) multiply(hh, hl, piece[u]);
    before();
    spill<LD>(hh, hl, sh.E + wave * TS * LD, f);
    __syncthreads();
  }
};
template <typename C, typename D>
union Either {
  typename C::Shared one;
  typename D::Shared other;
};
template <int TS>
using Core = std::conditional_t<TS == 128, Core128, Core64<4>>;
template <typename C>
using Quarter = std::conditional_t<C::TS == 128, Core64<4>, C>;  // what works on 64 x 64 in the same workgroup

// A from ROWS rows of a tile in shared memory
template <int ROWS, int TS, int PARTS, int THREADS>
__device__ __forceinline__ void store_gram(float* E, int np, const Area& o, int i0, int j0, bool diagonal) {
  _Float16* a = o.sq + SQ_A * o.na;
  rows8<ROWS, TS, TS + 1, PARTS, THREADS>(E, [&](int r, int c, float (&v)[8]) {
    if (diagonal)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + r == j0 + c + k) o.diag[SQ_A * np + i0 + r] = v[k] * (1.f / SCALE), v[k] = 0.f;
    store8(a + place(i0 + r, j0 + c, np), v);
  });
  if (!diagonal) {
    __syncthreads();
    store_turned<ROWS, TS, TS + 1, THREADS>(E, a, np, j0, i0);
  }
}
// A = X X^t: a tile on or above the diagonal, or one part of its sum, which ortho_sum_kernel adds up in their order.
// (Adding them in the workgroup that ends last needs the other workgroups' tiles flushed through the XCDs' caches: 160 us
// where this and the launch behind it take 17, at eight 256 x 2304 matrices.)
template <typename C>
__device__ __forceinline__ void gram_tile(typename C::Shared& sh, const Tile& w, const Area& o, float* parts, int kc) {
  constexpr int TS = C::TS;
  const int i0 = w.i * TS, j0 = w.j * TS;
  const int k0 = w.split * kc, k1 = k0 + kc < w.mp ? k0 + kc : w.mp;
  C::run(sh, o.x, i0, w.mp, o.x, j0, w.mp, k0, k1, 1.f / SCALE, [] {});
  if (w.splits > 1) {
    float* mine = parts + w.part;
#pragma unroll 4
    for (int q = threadIdx.x; q < TS * TS; q += C::THREADS) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < C::PARTS; ++k) v += sh.E[k * TS * (TS + 1) + q / TS * (TS + 1) + q % TS];
      mine[q] = v;
    }
    return;
  }
  store_gram<TS, TS, C::PARTS, C::THREADS>(sh.E, w.np, o, i0, j0, w.i == w.j);
}
// 32 rows of a tile of A from its parts
template <int TS, int THREADS>
__device__ __forceinline__ void sum_tile(float* E, const Tile& w, const Area& o, const float* parts, int slice) {
  const float* mine = parts + w.part + slice * TS;
#pragma unroll
  for (int q = threadIdx.x * 4; q < 32 * TS; q += THREADS * 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < w.splits; ++s) {
      const float4 u = *reinterpret_cast<const float4*>(mine + (size_t)s * (TS * TS) + q);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    float* e = E + q / TS * (TS + 1) + q % TS;
    e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
  }
  __syncthreads();
  store_gram<32, TS, 1, THREADS>(E, w.np, o, w.i * TS + slice, w.j * TS, w.i == w.j);
}
template <int TS>
__global__ __launch_bounds__(256) void ortho_sum_kernel(Chain l, _Float16* base, const float* __restrict__ parts) {
  __shared__ float E[32 * (TS + 1)];
  const Tile w = l.gram[blockIdx.x];
  if (w.split || w.splits == 1) return;
  sum_tile<TS, 256>(E, w, Area(base, w, l.rect_ts, 0), parts, blockIdx.y * 32);
}

// out = q I + l G + f (G - tg I) (H - th I) + m M of symmetric matrices that commute (all are polynomials of one): a tile on
// or above the diagonal.  The scales of what is stored are in the factors of what lies off the diagonal:
// out_ij = fh g_i H_ij + (fg h_j + lo) G_ij + mo M_ij + fs sum, with g = diag G - tg, h = diag H - th.  M where ADD.
struct Stored {
  int at;       // which array
  float scale;  // what its entries off the diagonal are multiplied by
};
struct Op {
  int out, g, h, m;
  float tg, th, q, l, f, md, fg, fh, fs, lo, mo, back;  // back: one over out's scale
  Op() = default;
  Op(Stored o, Stored a, float ta, Stored b, float tb, float factor)
      : out(o.at), g(a.at), h(b.at), m(a.at), tg(ta), th(tb), q(0.f), l(0.f), f(factor), md(0.f), fg(factor * (o.scale / a.scale)),
        fh(factor * (o.scale / b.scale)), fs(factor * (o.scale / (a.scale * b.scale))), lo(0.f), mo(0.f), back(1.f / o.scale) {}
  Op plus(Stored o, float factor, Stored matrix) const {
    Op r = *this;
    r.m = matrix.at, r.md = factor, r.mo = factor * (o.scale / matrix.scale);
    return r;
  }
};
template <typename C, bool ADD>
__device__ __forceinline__ void square_tile(typename C::Shared& sh, const Tile& w, const Area& o, const Op& op) {
  constexpr int TS = C::TS;
  const int i0 = w.i * TS, j0 = w.j * TS;
  const _Float16 *g = o.sq + op.g * o.na, *h = o.sq + op.h * o.na;
  const float *gd = o.diag + op.g * w.np, *hd = o.diag + op.h * w.np;
  const _Float16* m = o.sq + op.m * o.na;
  struct Loaded {
    Both g, h, m;
    float gi, mi, hj[8];
  };
  const auto load = [&](int r, int c) {
    const size_t at = place(i0 + r, j0 + c, w.np);
    Loaded d;
    d.g = load8(g + at), d.h = load8(h + at), d.gi = gd[i0 + r];
    if constexpr (ADD) d.m = load8(m + at), d.mi = o.diag[op.m * w.np + i0 + r];
    *reinterpret_cast<float4*>(d.hj) = *reinterpret_cast<const float4*>(hd + j0 + c);
    *reinterpret_cast<float4*>(d.hj + 4) = *reinterpret_cast<const float4*>(hd + j0 + c + 4);
    return d;
  };
  Rows<C, decltype(load)> rows{load};
  C::run(sh, g, i0, w.np, h, j0, w.np, 0, w.np, 1.f, [&] { rows.fetch(0); });
  _Float16* out = o.sq + op.out * o.na;
  const bool diagonal = w.i == w.j;
  rows.run(sh.E, [&](int r, int c, float (&v)[8], const Loaded& d) {
    const int i = i0 + r, j = j0 + c;
    const float gi = op.fh * (d.gi - op.tg);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float hj = d.hj[k] - op.th;
      float e = fmaf(fmaf(op.fg, hj, op.lo), d.g[k], op.fs * v[k]);
      e = fmaf(gi, d.h[k], e);
      if constexpr (ADD) e = fmaf(op.mo, d.m[k], e);
      if (diagonal && i == j + k) {
        float y = fmaf(op.f * (d.gi - op.tg), hj, fmaf(op.l, d.gi, op.q)) + op.fs * op.back * v[k];
        if constexpr (ADD) y = fmaf(op.md, d.mi, y);
        o.diag[op.out * w.np + i] = y;
        e = 0.f;
      }
      v[k] = e;
    }
    store8(out + place(i, j, w.np), v);
  });
  if (!diagonal) {
    __syncthreads();
    store_turned<TS, TS, TS + 1, C::THREADS>(sh.E, out, w.np, j0, i0);
  }
}
// X <- R X of a tile, in shared memory; as the next X unless it is the LAST
template <typename C, bool LAST>
__device__ __forceinline__ void apply_tile(typename C::Shared& sh, const Tile& w, const Area& o, int R, float fs) {
  constexpr int TS = C::TS;
  const int i0 = w.i * TS, j0 = w.j * TS;
  const _Float16* a = o.sq + R * o.na;
  struct Loaded {
    Both x;
    float d;
  };
  const auto load = [&](int r, int c) { return Loaded{load8(o.x + place(i0 + r, j0 + c, w.mp)), o.diag[R * w.np + i0 + r]}; };
  Rows<C, decltype(load)> rows{load};
  const auto before = [&] { rows.fetch(0); };
  if constexpr (TS == 128) C::template run<true>(sh, a, i0, w.np, o.x, j0, w.mp, 0, w.np, fs, before);
  else C::run(sh, a, i0, w.np, o.xt, j0, w.np, 0, w.np, fs, before);
  rows.run(sh.E, [&](int r, int c, float (&v)[8], const Loaded& d) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = fmaf(d.d, d.x[k], v[k]);
    if constexpr (!LAST) store8(o.next + place(i0 + r, j0 + c, w.mp), v);
  });
  __syncthreads();
  if constexpr (!LAST && TS == 64) store_turned<TS, TS, TS + 1, C::THREADS>(sh.E, o.next_t, w.np, j0, i0);
}
// The last one's to the caller, as the result or into the weights
template <typename T, int TS>
__device__ __forceinline__ void hand_over(const float* E, const Mat& t, int i0, int j0, int update, float decay) {
  T* out = static_cast<T*>(t.dst);
  callers<TS, 8>(
      t, i0, j0,
      [&](auto N, size_t at, int many) {  // (the weights, inside or not: eight loads on their way)
        Few<T, N()> x{};
        if (update) x = load_few<T, N()>(out + whole(N, at, many));
        return x;
      },
      [&](auto N, size_t at, int many, int r, int c, bool tall, const auto& was) {
        Few<T, N()> x = was, y;
        to_front(N, x.v, many);
#pragma unroll
        for (int k = 0; k < N(); ++k) {
          const float v = E[(tall ? r + k : r) * (TS + 1) + (tall ? c : c + k)] * (1.f / SCALE);
          y.v[k] = (T)(update ? fmaf(-t.rate, v, decay * (float)x.v[k]) : v);
        }
        if (many == N()) store_few(out + at, y);
        else if constexpr (decltype(N)::parts)
#pragma unroll
          for (int k = 0; k < N(); ++k)
            if (k < many) out[at + k] = y.v[k];
      });
}

// A launch of one chain takes a piece of the other along: the first `blocks` workgroups' work.  (The narrow matrices' chain
// has as many launches as the wide ones' and little work in each: a call for one head takes 309 us with that chain behind,
// 231 with it riding; the detector's 1218 and 1100, the ragged list 373 and 268.)
enum { RIDE_GRAM, RIDE_SUM, RIDE_POLY, RIDE_APPLY };
struct Rider {
  const Tile* list;
  unsigned blocks;
  int what, from, kc;
  Op op;  // RIDE_POLY
};
template <typename C>
__device__ __forceinline__ void ride(typename C::Shared& sh, const Rider& r, _Float16* base, float* parts) {
  static_assert(C::TS == 64, "the chain that rides is in tiles of 64");
  const bool sum = r.what == RIDE_SUM;
  const Tile w = r.list[sum ? blockIdx.x / 2 : blockIdx.x];
  const Area o(base, w, 64, r.from);
  if (r.what == RIDE_GRAM) gram_tile<C>(sh, w, o, parts, r.kc);
  else if (r.what == RIDE_POLY) square_tile<C, false>(sh, w, o, r.op);
  else if (r.what == RIDE_APPLY) apply_tile<C, false>(sh, w, o, r.op.out, 1.f / SCALE);
  else if (w.split == 0 && w.splits > 1) sum_tile<64, C::THREADS>(sh.E, w, o, parts, blockIdx.x % 2 * 32);
}

template <int TS, bool RIDE>
__global__ __launch_bounds__(256, 2) void ortho_gram_kernel(Chain l, Rider r, _Float16* base, float* parts, int kc, int from) {
  __shared__ Either<Core<TS>, Core64<4>> sh;
  if constexpr (RIDE)
    if (blockIdx.x < r.blocks) return ride<Core64<4>>(sh.other, r, base, parts);
  const Tile w = l.gram[blockIdx.x - (RIDE ? r.blocks : 0)];
  const Area o(base, w, l.rect_ts, from);
  if (w.ts == TS) gram_tile<Core<TS>>(sh.one, w, o, parts, kc);
  if constexpr (TS == 128)
    if (w.ts == 64) gram_tile<Core64<4>>(sh.other, w, o, parts, kc);
}
template <typename C, bool ADD, bool RIDE>
__global__ __launch_bounds__(C::THREADS, 2) void ortho_square_kernel(Chain l, Rider r, _Float16* base, float* parts, Op first,
                                                                     Op second) {
  __shared__ Either<C, Quarter<C>> sh;
  if constexpr (RIDE)
    if (blockIdx.x < r.blocks) {
      if (blockIdx.y == 0) ride<Quarter<C>>(sh.other, r, base, parts);
      return;
    }
  const Tile w = l.tri[blockIdx.x - (RIDE ? r.blocks : 0)];
  const Area o(base, w, l.rect_ts, 0);
  const Op op = blockIdx.y ? second : first;
  if (w.ts == C::TS) square_tile<C, ADD>(sh.one, w, o, op);
  if constexpr (C::TS == 128)
    if (w.ts == 64) square_tile<Core64<4>, ADD>(sh.other, w, o, op);
}
template <int TS, bool RIDE>
__global__ __launch_bounds__(256, 2) void ortho_apply_kernel(Chain l, Rider r, _Float16* base, float* parts, int R, float fs,
                                                             int from) {
  __shared__ Either<Core<TS>, Core64<4>> sh;
  if constexpr (RIDE)
    if (blockIdx.x < r.blocks) return ride<Core64<4>>(sh.other, r, base, parts);
  const Tile w = l.rect[blockIdx.x - (RIDE ? r.blocks : 0)];
  apply_tile<Core<TS>, false>(sh.one, w, Area(base, w, TS, from), R, fs);
}
struct Product {  // what the last X is made of
  int R, from;
  float fs;
};
// (the other chain's tiles, of 64, are the first `others`)
template <typename T, int TS>
__global__ __launch_bounds__(256, 2) void ortho_apply_last_kernel(const Mat* table, Chain l, Product p, const Tile* other,
                                                            unsigned others, Product q, _Float16* base, int update, float decay) {
  __shared__ Either<Core<TS>, Core64<4>> sh;
  if (blockIdx.x < others) {
    const Tile w = other[blockIdx.x];
    apply_tile<Core64<4>, true>(sh.other, w, Area(base, w, 64, q.from), q.R, q.fs);
    hand_over<T, 64>(sh.other.E, table[w.mat], w.i * 64, w.j * 64, update, decay);
    return;
  }
  const Tile w = l.rect[blockIdx.x - others];
  apply_tile<Core<TS>, true>(sh.one, w, Area(base, w, TS, p.from), p.R, p.fs);
  hand_over<T, TS>(sh.one.E, table[w.mat], w.i * TS, w.j * TS, update, decay);
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix of at most 64 x 128 stays in one workgroup's shared memory from the first step to the last, so that a list of such
// is one launch instead of two dozen that wait for each other (64 x 64: 15 us against 127).  One step at a time: X and X^t,
// A and F, each 16 x 16 of a product a wavefront (sixteen; four of 32 x 32 wait for each instruction by themselves: 23 us).
// A lane holds four neighbouring entries of a column of the product, which are four of a row of X^t, or of A and F, which
// are symmetric.
constexpr int SMALL_N = 64, SMALL_M = 128, SMALL_THREADS = 1024;
__host__ __device__ inline bool is_small(int rows, int cols) {
  return (rows < cols ? rows : cols) <= SMALL_N && (rows < cols ? cols : rows) <= SMALL_M;
}
struct Small {
  _Float16 x[SMALL_M / 32 * BLOCK], xt[SMALL_M / 32 * BLOCK], a[2 * BLOCK], f[2 * BLOCK];
  float da[64], df[64];
  double norm[SMALL_THREADS / 64];
};
// 16 x 16 at (i, j) of P Q^t over K columns, which both have
template <int K>
__device__ __forceinline__ float4v small_product(const _Float16* p, int i, const _Float16* q, int j) {
  float4v hh = {}, hl = {}, lh = {};
  const int lane = threadIdx.x & 63, r = lane & 15, c = 8 * (lane >> 4);
  half8 ph[K / 32], pl[K / 32], qh[K / 32], ql[K / 32];
#pragma unroll
  for (int k = 0; k < K / 32; ++k) {
    const _Float16 *u = p + place(i + r, k * 32 + c, K), *v = q + place(j + r, k * 32 + c, K);
    ph[k] = *reinterpret_cast<const half8*>(u), pl[k] = *reinterpret_cast<const half8*>(u + LO);
    qh[k] = *reinterpret_cast<const half8*>(v), ql[k] = *reinterpret_cast<const half8*>(v + LO);
  }
#pragma unroll
  for (int k = 0; k < K / 32; ++k) {  // (three chains: a matrix instruction waits for the one before it on the same sum)
    hh = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[k], qh[k], hh, 0, 0, 0);
    hl = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[k], ql[k], hl, 0, 0, 0);
    lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[k], qh[k], lh, 0, 0, 0);
  }
  return hh + (hl + lh);
}
__device__ __forceinline__ void put4(_Float16* at, const float (&v)[4]) {
  half4 h, l;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    _Float16 hh, ll;
    split16(v[k], hh, ll);
    h[k] = hh, l[k] = ll;
  }
  *reinterpret_cast<half4*>(at) = h;
  *reinterpret_cast<half4*>(at + LO) = l;
}
__device__ __forceinline__ void get4(float (&v)[4], const _Float16* at) {
  const half4 h = *reinterpret_cast<const half4*>(at), l = *reinterpret_cast<const half4*>(at + LO);
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = (float)h[k] + (float)l[k];
}
struct Step {  // F = q I + l A + c (A - t I)^2
  float c, t, q, l;
};
template <typename T, int mp>
__device__ __forceinline__ void small_matrix(Small& sh, const Mat& t, const Momentum& m, const Step& p, int steps, double eps,
                                             float decay) {
  const bool tall = t.rows > t.cols;
  const int shift = tall || mp == 64 ? 6 : 7;  // of the columns of the padded matrix as the caller has it
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  {
    constexpr int EACH = SMALL_N * mp / SMALL_THREADS;
    float v[EACH], u[EACH];
    double s = 0;
    const auto at = [&](int k, bool& in) {
      const int e = k * SMALL_THREADS + threadIdx.x, r = e >> shift, c = e & ((1 << shift) - 1);
      in = r < t.rows && c < t.cols;
      return in ? (size_t)r * t.cols + c : 0;
    };
    bool in;  // (every load before the first use, inside or not)
#pragma unroll
    for (int k = 0; k < EACH; ++k) v[k] = (float)static_cast<const T*>(t.src)[at(k, in)];
    if (m.update) {
#pragma unroll
      for (int k = 0; k < EACH; ++k) u[k] = t.buf[at(k, in)];
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const size_t where = at(k, in);
      if (m.update) {
        u[k] = fmaf(m.mu, u[k], v[k]);
        if (in) t.buf[where] = u[k];
        v[k] = m.nesterov ? fmaf(m.mu, u[k], v[k]) : u[k];
      }
      v[k] = in ? v[k] : 0.f;
      s = fma((double)v[k], (double)v[k], s);
    }
    s = block_sum<SMALL_THREADS>(s, sh.norm);
    const double inv = (double)SCALE / (sqrt(s) + eps);
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int e = k * SMALL_THREADS + threadIdx.x, r = e >> shift, c = e & ((1 << shift) - 1);
      const int i = tall ? c : r, j = tall ? r : c;
      _Float16 h, l;
      split16((float)((double)v[k] * inv), h, l);
      const size_t x = place(i, j, mp), y = place(j, i, 64);
      sh.x[x] = h, sh.x[x + LO] = l, sh.xt[y] = h, sh.xt[y + LO] = l;
    }
  }
  __syncthreads();
  // this wavefront's 16 x 16 begin at (i, j); this lane's four at row r of column c
  const int i = (wave >> 2) * 16, j = (wave & 3) * 16, r = i + 4 * (lane >> 4), c = j + (lane & 15);
  T* out = static_cast<T*>(t.dst);
  const auto target = [&](int a, int b, bool& in) {
    const int row = tall ? b : a, col = tall ? a : b;
    in = row < t.rows && col < t.cols;
    return in ? (size_t)row * t.cols + col : 0;
  };
  T was[mp / 64][4];  // the weights: on their way while the steps are taken
  if (m.update) {
    bool in;
#pragma unroll
    for (int h = 0; h < mp / 64; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k) was[h][k] = out[target(r + k, c + 64 * h, in)];
  }
  float v[mp / 64][4];
  const int diagonal = c - r;  // the place of this column's diagonal entry among the four, if it is one of them
  const bool has = diagonal >= 0 && diagonal < 4;
  for (int step = 0;; ++step) {
    {
      const float4v acc = small_product<mp>(sh.x, i, sh.x, j);
      float a[4], d = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = acc[k] * (1.f / SCALE);
        d = diagonal == k ? a[k] : d;
        a[k] = diagonal == k ? 0.f : a[k];
      }
      put4(sh.a + place(c, r, 64), a);
      if (has) sh.da[c] = d * (1.f / SCALE);
    }
    __syncthreads();
    {
      const float4v acc = small_product<64>(sh.a, i, sh.a, j);
      const float aj = sh.da[c], dj = aj - p.t, cs = p.c / SCALE;
      float a[4], d = 0.f;
      get4(a, sh.a + place(c, r, 64));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float sum = cs * acc[k];
        a[k] = fmaf(fmaf(p.c, sh.da[r + k] - p.t + dj, p.l), a[k], sum);
        d = diagonal == k ? sum : d;
        a[k] = diagonal == k ? 0.f : a[k];
      }
      put4(sh.f + place(c, r, 64), a);
      if (has) sh.df[c] = fmaf(p.c * dj, dj, fmaf(p.l, aj, p.q)) + d * (1.f / SCALE);
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < mp / 64; ++h) {
      const float4v acc = small_product<64>(sh.f, i, sh.xt, j + 64 * h);
      float x[4];
      get4(x, sh.xt + place(c + 64 * h, r, 64));
#pragma unroll
      for (int k = 0; k < 4; ++k) v[h][k] = fmaf(sh.df[r + k], x[k], acc[k] * (1.f / SCALE));
    }
    if (step + 1 == steps) break;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < mp / 64; ++h) {
      half4 hi, lo;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        _Float16 u, w;
        split16(v[h][k], u, w);
        hi[k] = u, lo[k] = w;
      }
      _Float16* at = sh.xt + place(c + 64 * h, r, 64);
      *reinterpret_cast<half4*>(at) = hi;
      *reinterpret_cast<half4*>(at + LO) = lo;
      at = sh.x + place(r, c + 64 * h, mp);  // (rows of eight columns lie behind each other: r + 1 is 8 further)
#pragma unroll
      for (int k = 0; k < 4; ++k) at[8 * k] = hi[k], at[8 * k + LO] = lo[k];
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < mp / 64; ++h)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      bool in;
      const size_t at = target(r + k, c + 64 * h, in);
      const float y = v[h][k] * (1.f / SCALE);
      if (in) out[at] = (T)(m.update ? fmaf(-t.rate, y, decay * (float)was[h][k]) : y);
    }
}
template <typename T>
__global__ __launch_bounds__(SMALL_THREADS) void ortho_small_kernel(Batch b, Momentum m, Step p, int steps, double eps, float decay) {
  __shared__ Small sh;
  const Mat t = b.m[blockIdx.x];
  if (t.rows <= 64 && t.cols <= 64) small_matrix<T, 64>(sh, t, m, p, steps, eps, decay);
  else small_matrix<T, 128>(sh, t, m, p, steps, eps, decay);
}

// ------------------------------------------------------------------------------------------------ the host
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

// Matrices are taken in chains of launches by what their accuracy allows.  In a group of steps the next A is made of products,
// whose roundings the largest singular value carries over into the smallest ones' directions, where every later step
// multiplies them by a a: with one value 12 to 40 times the others, groups of 3 + 2 leave an error of 56e-6 with 2 rows, 50e-6
// with 5, 15e-6 with 65, 14e-6 with 135, 10e-6 with 192, 7e-6 with 256 (any columns), where the form op by op in fp32 has
// 2e-6, 2e-6, 3e-6, 4e-6, 6e-6 and 8e-6, and single steps 1e-6 throughout.  So from NARROW rows on groups are no worse than
// that form at its worst, and matrices of fewer take single steps whatever else is in the list.
constexpr int NARROW = 256;
enum { SMALLS = 1, NARROWS = 2, WIDES = 4 };
int kind(int rows, int cols) {
  return is_small(rows, cols) ? SMALLS : (rows < cols ? rows : cols) < NARROW ? NARROWS : WIDES;
}
// a list that is taken
bool taken(int count, const int* rows, const int* cols) {
  if (count < 0 || count > (1 << 16) || (count && (!rows || !cols))) return false;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 1 || cols[i] < 1 || (int64_t)rows[i] * cols[i] > 0x7fffffff) return false;
    if ((rows[i] < cols[i] ? rows[i] : cols[i]) > 32768) return false;
    if ((rows[i] > cols[i] ? rows[i] : cols[i]) > 65535 * 64) return false;  // (a tile's place has 16 bits)
  }
  return true;
}
// One chain of launches: the matrices of some kinds.
struct Work {
  int kinds;
  bool single;  // steps one by one
  int kc;       // the summed index of X X^t a workgroup takes at most
  bool split;   // whether any matrix has more than one part
  int narrow;   // the smallest n
  unsigned count;
  uint64_t part, halves, fill, elements;
  Chain c;      // (sizes only)
  unsigned parts_of(const Dim& d) const { return (unsigned)((d.mp + kc - 1) / kc); }
};
// 0: fine, -1: too many tiles
int work(int count, const int* rows, const int* cols, int kinds, Work& p) {
  const auto skip = [&](int i) { return !(kind(rows[i], cols[i]) & kinds); };
  p = Work{};
  p.kinds = kinds;
  p.narrow = 1 << 30;
  Chain& l = p.c;
  // Tiles: 128 needs half the reads of two operands that 64 does, and is taken for a pass that fills the card with such
  // tiles; X X^t, in parts, and R X, with short sums, from half of that on.  The n x n products: at 528 tiles of 128
  // (4096 x 4096, none quartered) 273 us, 307 with four times as many of 64; at 292 (the detector's) 45, 35 so.  R X at
  // 2616: 184 us, 256 so; at 256 (2048 x 2048) 70, 71.  X X^t at 730 parts: 95 + 17 us, 113 + 6 so.
  uint64_t tri128 = 0, rect128 = 0, gram128 = 0;
  for (int i = 0; i < count; ++i) {
    if (skip(i)) continue;
    ++p.count;
    const Dim w(rows[i], cols[i]);
    if (w.n < p.narrow) p.narrow = w.n;
    p.elements += (uint64_t)rows[i] * cols[i];
    tri128 += w.tri(128), rect128 += w.rect(128);
    gram128 += (uint64_t)w.tri(128) * ((w.mp + 255) / 256);
  }
  l.gram_ts = gram128 >= WANT / 2 ? 128 : 64;
  l.tri_ts = tri128 >= WANT ? 128 : 64;
  l.rect_ts = rect128 >= WANT / 2 ? 128 : 64;
  // Whole tiles fill the card so many times; a few that are left would each keep a compute unit for a tile's time, alone,
  // and are quartered (16 of 528, 4096 x 4096: an n x n product 275 -> 234 us, X X^t 255 -> 222).
  const auto quarter = [](uint64_t& n, bool big) {
    const unsigned rest = big && n >= WANT && n % WANT <= WANT / 4 ? (unsigned)(n % WANT) : 0;
    const unsigned whole = (unsigned)n - rest;
    n = whole + 4 * (uint64_t)rest;
    return whole;
  };
  // X X^t: how much of its sum a workgroup takes.  In stages' times: the card takes WANT workgroups at a time, with some 8
  // in front of and behind their own; where there are parts, their sums are a launch (4) and pass over them (60 tiles of 128
  // a stage).  (2048 x 2048: parts of 768, 41 + 11 us; of 512, 44 + 11.  The detector's: 768 too, 89 + 20; of 1024,
  // 98 + 16; of 2048, 104 + 11.  4096 x 4096: whole, 222; of 1024, 231 + 38.)
  uint64_t least = ~0ull;
  for (int kc = 4096; kc >= 512; kc -= 128) {
    uint64_t blocks = 0, whole = 0;
    for (int i = 0; i < count; ++i) {
      if (skip(i)) continue;
      const Dim d(rows[i], cols[i]);
      blocks += (uint64_t)d.tri(l.gram_ts) * ((d.mp + kc - 1) / kc), whole += d.tri(l.gram_ts);
    }
    const bool split = blocks > whole;
    if (!split) blocks = quarter(blocks, l.gram_ts == 128);  // (the quarters are done by the way)
    const uint64_t cost = (blocks + WANT - 1) / WANT * (kc / 32 + 8) + (split ? 4 + blocks / (l.gram_ts == 128 ? 60 : 240) : 0);
    if (cost <= least) least = cost, p.kc = kc;
  }
  uint64_t gram = 0, tri = 0, rect = 0;
  for (int i = 0; i < count; ++i) {
    if (skip(i)) continue;
    const Dim d(rows[i], cols[i]);
    const unsigned s = p.parts_of(d);
    gram += (uint64_t)d.tri(l.gram_ts) * s;
    tri += d.tri(l.tri_ts);
    rect += d.rect(l.rect_ts);
    p.fill += d.rect(64);
    if (s > 1) p.part += (uint64_t)d.tri(l.gram_ts) * s * l.gram_ts * l.gram_ts, p.split = true;
    p.halves += d.halves(l.rect_ts);
  }
  l.whole_gram = quarter(gram, l.gram_ts == 128 && !p.split), l.whole_tri = quarter(tri, l.tri_ts == 128);
  const uint64_t most = (1 << 23) - 1;  // (a launch has fewer than 2^32 threads: two chains' tiles by 256)
  if (gram > most || tri > most || rect > most || p.fill > most) return -1;  // (workspaces of 274 GB and more)
  l.n_gram = (unsigned)gram, l.n_tri = (unsigned)tri, l.n_rect = (unsigned)rect;
  return 0;
}
// Where every pass has at most a tile a compute unit, the two passes over X are launches like the others: steps are taken
// one by one, if X X^t is a launch as well (250 x 250: 104 us, 111 in groups; 300 x 300: 117, 126) or a matrix is narrow.
bool one_by_one(const Work& p) {
  const Chain& l = p.c;
  return l.gram_ts == 64 && l.tri_ts == 64 && l.rect_ts == 64 && l.n_gram <= CARD && l.n_tri <= CARD && l.n_rect <= CARD &&
         (!p.split || p.narrow < NARROW);
}

// The whole list: all but the small matrices in one chain, in single steps, where that is as fast; else the wide ones in
// groups and the narrow ones in single steps.  Every part of the workspace is a multiple of 256 bytes.
struct Plan {
  size_t table, gram[2], tri[2], rect[2], fill, norm_map, norms, parts, halves, total;
  Lists l;  // (sizes only)
  Work w[2];
  int chains;
};
// 0: fine, -1: a list that is not taken
int plan(int count, const int* rows, const int* cols, Plan& p) {
  p.chains = 0, p.total = 256;  // (nothing but small matrices needs nothing)
  p.w[0].single = false;
  if (!taken(count, rows, cols)) return -1;
  int kinds = 0;
  uint64_t tiles = 0;  // (of 64)
  for (int i = 0; i < count; ++i) {
    const int k = kind(rows[i], cols[i]) & (NARROWS | WIDES);
    kinds |= k;
    if (k) tiles += Dim(rows[i], cols[i]).rect(64);
  }
  if (!kinds) return 0;
  const bool both = kinds == (NARROWS | WIDES);
  p.chains = 1;
  if (!both || tiles <= CARD) {  // (more are not taken one by one)
    if (work(count, rows, cols, kinds, p.w[0]) != 0) return -1;
    p.w[0].single = kinds == NARROWS || one_by_one(p.w[0]);
  }
  if (both && !p.w[0].single) {
    if (work(count, rows, cols, WIDES, p.w[0]) != 0 || work(count, rows, cols, NARROWS, p.w[1]) != 0) return -1;
    p.w[1].single = true;
    p.chains = 2;
  }
  Lists& l = p.l;
  l = Lists{};
  uint64_t elements = 0, norm = 0, fill = 0, part = 0, halves = 0, entries = 0;
  for (int k = 0; k < p.chains; ++k) elements += p.w[k].elements;
  // The norms: each thread 32 elements, fewer where that would leave compute units without work (2.6 M elements: 20 us, 6 so).
  for (l.chunk = 8192; l.chunk > 1024 && elements / l.chunk < 2 * WANT;) l.chunk /= 2;
  for (int i = 0; i < count; ++i)
    if (kind(rows[i], cols[i]) != SMALLS) norm += Dim(rows[i], cols[i]).norms(l.chunk);
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t was = at;
    at += round256(bytes);
    return was;
  };
  for (int k = 0; k < p.chains; ++k) {
    const Work& w = p.w[k];
    fill += w.fill, part += w.part, halves += w.halves;
    entries += (uint64_t)w.c.n_gram + w.c.n_tri + w.c.n_rect;
    p.gram[k] = take(sizeof(Tile) * (size_t)w.c.n_gram);
    p.tri[k] = take(sizeof(Tile) * (size_t)w.c.n_tri);
    p.rect[k] = take(sizeof(Tile) * (size_t)w.c.n_rect);
  }
  if (entries + fill + norm > 0x7fffffff) return -1;  // (of the lists' kernel)
  l.n_fill = (unsigned)fill, l.n_norm = (unsigned)norm;
  l.second = p.w[0].count;
  p.table = take(sizeof(Mat) * (size_t)(p.w[0].count + (p.chains > 1 ? p.w[1].count : 0)));
  p.fill = take(sizeof(Tile) * fill);
  p.norm_map = take(sizeof(uint2) * norm);
  p.norms = take(sizeof(double) * norm);
  p.parts = take(sizeof(float) * part);
  p.halves = take(sizeof(_Float16) * halves);
  p.total = at;
  return 0;
}

// How a step's polynomial is taken: F = q I + l A + c (A - t I)^2.  The square is completed (l = 0) unless that needs large
// numbers (c near 0): then t = 0.
struct Poly {
  float c, t, q, l;
  int longest;  // group; 0: an iterate might leave fp16's range
  bool brief;   // whether a group's steps can be taken in fewer launches: the products of that stay in range, too
};
// Groups of steps: twos, the first a three where the number is odd; ones where R of a longer group might leave its range
int group_length(int left, int steps) { return left == 1 ? 1 : (left == steps && left % 2 ? 3 : 2); }
// The spectral norms of X, A, F A, F off the diagonal from |X| <= 1 on, step by step, with the polynomials' extremes in
// between (1 % over, for the roundings).
Poly polynomial(int steps, double a, double b, double c) {
  Poly r{(float)c, 0.f, (float)a, (float)b, 0, false};
  if (!(fabs(a) < 1e6) || !(fabs(b) < 1e6) || !(fabs(c) < 1e6)) return r;
  const double most = 65504.0 / SCALE / 1.05;
  double t = 0, q = a, f = b;
  if (c != 0 && fabs(b) <= 14 * fabs(c)) {
    // t and c as they will be multiplied; q makes up for their rounding (a is the factor of what is far from 1 already:
    // 4.5 units of the last place off in every step otherwise)
    c = (float)c;
    t = (float)(-b / (2 * c)), q = a - c * t * t, f = 0;
  }
  double top = 1, high = 0, most_a = 0;  // the largest |X|, and |F| and |A| so far
  for (int k = 0; k < steps; ++k) {
    const auto X = [&](double s) { return fabs(s * (a + s * s * (b + s * s * c))); };
    const auto Q = [&](double v) { return a + v * (b + v * c); };
    const double t1 = top * top;
    double x = X(top), now = fmax(fabs(Q(0)), fabs(Q(t1))), e = fmax(fabs(Q(0) - q), fabs(Q(t1) - q));
    const double tb = c != 0 ? -b / (2 * c) : -1;  // where b + 2 c v = 0
    if (tb > 0 && tb < t1) now = fmax(now, fabs(Q(tb))), e = fmax(e, fabs(Q(tb) - q));
    // where a + 3 b v + 5 c v v = 0
    double z[2] = {-1, -1};
    if (c != 0) {
      const double w = 9 * b * b - 20 * a * c;
      if (w >= 0) z[0] = (-3 * b + sqrt(w)) / (10 * c), z[1] = (-3 * b - sqrt(w)) / (10 * c);
    } else if (b != 0) {
      z[0] = -a / (3 * b);
    }
    for (double v : z)
      if (v > 0 && v < t1) x = fmax(x, X(sqrt(v)));
    high = fmax(high, now), most_a = fmax(most_a, t1);
    if (!(t1 <= most) || !(x <= most) || !(x * top <= most) || !(e <= most)) return r;
    top = 1.01 * x;
  }
  r.t = (float)t, r.q = (float)q, r.l = (float)f;
  const double room = 65504.0 / R_SCALE / 1.05;  // R off its diagonal: that of R - q^g I
  q = fabs(q);
  r.longest = high * high * high + q * q * q <= room ? 3 : high * high + q * q <= room ? 2 : 1;
  r.brief = f == 0 && r.longest == 3 && high * high * (most_a + fabs(t)) <= room;
  return r;
}

template <typename F>
void choose(int ts, const F& f) {  // f(tile) with the tile a constant
  if (ts == 128) f(std::integral_constant<int, 128>());
  else f(std::integral_constant<int, 64>());
}

// The narrow chain's launches but its last, one after the other, for those of the wide one to take along.
struct Rides {
  const Chain* c;  // (null: none)
  int kc;
  bool split;
  int steps;  // that are left
  Op op;      // of its products
  int what = RIDE_GRAM, from = 0;
  bool left() const { return c && (steps > 1 || what != RIDE_APPLY); }
  Rider next() {
    if (!left()) return Rider{};
    Rider r{c->gram, c->n_gram, what, from, kc, op};
    if (what == RIDE_GRAM) {
      what = split ? RIDE_SUM : RIDE_POLY;
    } else if (what == RIDE_SUM) {
      r.blocks *= 2, what = RIDE_POLY;
    } else if (what == RIDE_POLY) {
      r.list = c->tri, r.blocks = c->n_tri, what = RIDE_APPLY;
    } else {
      r.list = c->rect, r.blocks = c->n_rect, what = RIDE_GRAM;
      from ^= 1, --steps;
    }
    return r;
  }
};

template <typename T>
int run(int count, const void* const* src, void* const* dst, float* const* buf, const int* rows, const int* cols,
        const float* rates, float decay, float mu, int nesterov, int steps, const Poly& f, double eps, const Plan& p, char* ws,
        hipStream_t st) {
  const int update = buf != nullptr;
  const Momentum m{update, nesterov, mu};
  const dim3 wg(256);
  const auto matrix = [&](int i) {
    return Mat{src[i], dst[i], update ? buf[i] : nullptr, rows[i], cols[i], rates ? rates[i] : 0.f, 1};
  };
  for (int i = 0; i < count;) {
    Batch batch{};
    for (; i < count && batch.count < BATCH; ++i)
      if (kind(rows[i], cols[i]) == SMALLS) batch.m[batch.count++] = matrix(i);
    if (batch.count)
      hipLaunchKernelGGL((ortho_small_kernel<T>), dim3(batch.count), dim3(SMALL_THREADS), 0, st, batch, m, Step{f.c, f.t, f.q, f.l}, steps, eps,
                         decay);
    if (hipGetLastError() != hipSuccess) return -2;
  }
  if (p.chains == 0) return 0;
  Lists lists = p.l;
  lists.table = reinterpret_cast<Mat*>(ws + p.table);
  lists.fill = reinterpret_cast<Tile*>(ws + p.fill);
  lists.norm_map = reinterpret_cast<uint2*>(ws + p.norm_map);
  for (int k = 0; k < p.chains; ++k) {
    lists.c[k] = p.w[k].c;
    lists.c[k].gram = reinterpret_cast<Tile*>(ws + p.gram[k]);
    lists.c[k].tri = reinterpret_cast<Tile*>(ws + p.tri[k]);
    lists.c[k].rect = reinterpret_cast<Tile*>(ws + p.rect[k]);
  }
  double* norms = reinterpret_cast<double*>(ws + p.norms);
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  _Float16* base = reinterpret_cast<_Float16*>(ws + p.halves);
  {
    Mat next{};  // (what the next matrix's entries begin at)
    if (p.chains > 1) {  // (the second chain's begin behind the first's, before those were quartered)
      Chain& c = lists.c[1];
      for (int i = 0; i < count; ++i) {
        if (!(kind(rows[i], cols[i]) & p.w[0].kinds)) continue;
        const Dim d(rows[i], cols[i]);
        c.gram0 += d.tri(lists.c[0].gram_ts) * p.w[0].parts_of(d), c.tri0 += d.tri(lists.c[0].tri_ts);
        c.rect0 += d.rect(lists.c[0].rect_ts);
      }
    }
    unsigned first = 0;
    Batch batch{};
    const auto flush = [&] {
      batch.end = next;
      const Mat& was = batch.m[0];
      const unsigned entries = next.gram0 - was.gram0 + (next.tri0 - was.tri0) + (next.rect0 - was.rect0) +
                               (next.fill0 - was.fill0) + (next.norm0 - was.norm0);
      hipLaunchKernelGGL(ortho_lists_kernel, dim3((entries + 255) / 256), wg, 0, st, lists, batch, first);
      first += batch.count;
      batch.count = 0;
    };
    for (int k = 0; k < p.chains; ++k)
      for (int i = 0; i < count; ++i) {
        const Work& w = p.w[k];
        if (!(kind(rows[i], cols[i]) & w.kinds)) continue;
        const Dim d(rows[i], cols[i]);
        Mat& t = batch.m[batch.count++];
        t = matrix(i);
        t.splits = w.parts_of(d);
        t.gram0 = next.gram0, t.tri0 = next.tri0, t.rect0 = next.rect0, t.fill0 = next.fill0, t.norm0 = next.norm0;
        t.part0 = next.part0, t.at = next.at;
        next.gram0 += d.tri(w.c.gram_ts) * t.splits;
        next.tri0 += d.tri(w.c.tri_ts);
        next.rect0 += d.rect(w.c.rect_ts);
        next.fill0 += d.rect(64);
        next.norm0 += d.norms(lists.chunk);
        if (t.splits > 1) next.part0 += (size_t)d.tri(w.c.gram_ts) * t.splits * w.c.gram_ts * w.c.gram_ts;
        next.at += d.halves(w.c.rect_ts);
        if (batch.count == BATCH) flush();
      }
    if (batch.count) flush();
    if (hipGetLastError() != hipSuccess) return -2;
  }
  hipLaunchKernelGGL((ortho_norm_kernel<T>), dim3(lists.n_norm), wg, 0, st, lists, norms, m);
  hipLaunchKernelGGL((ortho_start_kernel<T>), dim3(lists.n_fill), wg, 0, st, lists, norms, base, m, eps);
  if (hipGetLastError() != hipSuccess) return -2;
  const unsigned cus = (unsigned)r3_cu_count();
  const auto polynomial_of = [&](Stored out, Stored a) {
    Op r(out, a, f.t, a, f.t, f.c);
    r.q = f.q, r.l = f.l, r.lo = f.l * (out.scale / a.scale);
    return r;
  };
  const auto times = [](Stored out, Stored g, Stored h) { return Op(out, g, 0.f, h, 0.f, 1.f); };
  const auto of_step = [&] { return polynomial_of(Stored{SQ_F, SCALE}, Stored{SQ_A, SCALE}); };
  // The narrow chain rides where it is in tiles of 64 throughout (one in larger ones has work for the card by itself).
  const Chain& second = lists.c[1];
  const bool riding = p.chains > 1 && second.gram_ts == 64 && second.tri_ts == 64 && second.rect_ts == 64;
  Rides rides{riding ? &second : nullptr, p.w[1].kc, p.w[1].split, steps, of_step()};
  const auto chain = [&](const Chain& l, const Work& w) {
  const auto square = [&](const Op& one, const Op* two, bool add = false) {
    const Rider r = rides.next();
    const dim3 grid(r.blocks + l.n_tri, two ? 2 : 1);
    const auto launch_as = [&](auto core, auto ADD, auto RIDE) {
      typedef decltype(core) C;
      hipLaunchKernelGGL((ortho_square_kernel<C, ADD(), RIDE()>), grid, dim3(C::THREADS), 0, st, l, r, base, parts, one,
                         two ? *two : one);
    };
    const auto launch = [&](auto core, auto ADD) {
      if (r.blocks) launch_as(core, ADD, std::true_type());
      else launch_as(core, ADD, std::false_type());
    };
    // A tile a compute unit: eight wavefronts share its sum and its epilogue (eight of 256 x 256: 7.3 us, four 8.4; more
    // tiles than that share the units anyway: 2048 x 2048, 56 against 53).
    const bool eight = r.blocks + l.n_tri * grid.y <= cus;
    if (l.tri_ts == 128) launch(Core128(), std::false_type());
    else if (add && eight) launch(Core64<8>(), std::true_type());
    else if (add) launch(Core64<4>(), std::true_type());
    else if (eight) launch(Core64<8>(), std::false_type());
    else launch(Core64<4>(), std::false_type());
  };
  const auto both = [&](const Op& one, const Op& two, bool add = false) { square(one, &two, add); };
  // R of a group of g steps, in launches of at most two products
  const auto group = [&](int g) {
    const Stored A{SQ_A, SCALE}, FA{SQ_FA, SCALE};
    Stored R{SQ_F, SCALE}, spare{SQ_R, R_SCALE};
    for (int k = 0; k < g; ++k) {
      const Stored F{SQ_F + (k & 1), SCALE};
      square(polynomial_of(F, A), nullptr);
      if (k) {
        const Op next = times(spare, F, R);
        if (k + 1 < g) both(next, times(FA, F, A));
        else square(next, nullptr);
        R = spare, spare.at = SQ_R + (R.at == SQ_R);
      } else if (k + 1 < g) {
        square(times(FA, F, A), nullptr);
      }
      if (k + 1 < g) square(times(A, F, FA), nullptr);
    }
    return R;
  };
  // The same in one launch less for every step but the first, with a product more: where two products' tiles find a compute
  // unit each, a launch is what counts (one head: 79 us of products, 86 as above; 1025 x 511: 96, 110).  With A' = F F A, the
  // next step's A, and R so far:
  //   A' R = (F A) (F R),  H = A' R - t R,  and the next R = F(A') R = q R + c (A' - t I) H.
  const auto brief_group = [&](int g) {
    const Stored A{SQ_A, SCALE}, FA{SQ_FA, SCALE};
    Stored F{SQ_F, SCALE}, R = F, FR{SQ_R + 1, R_SCALE}, H{SQ_F + 1, R_SCALE}, next{SQ_R, R_SCALE};
    square(polynomial_of(F, A), nullptr);
    for (int k = 1; k < g; ++k) {
      both(times(FA, F, A), times(FR, F, R));
      both(times(A, F, FA), times(H, FA, FR).plus(H, -f.t, R), true);
      const Op step = Op(next, A, f.t, H, 0.f, f.c).plus(next, f.q, R);
      const Stored was = F;
      if (k + 1 < g) {
        F = Stored{FR.at, SCALE};
        both(step, polynomial_of(F, A), true);
        R = next, FR = Stored{was.at, R_SCALE}, next = Stored{F.at, R_SCALE};
      } else {
        square(step, nullptr, true);
        R = next;
      }
    }
    return R;
  };
  const bool brief = f.brief && l.tri_ts == 64 && 2 * l.n_tri <= cus;
  int from = 0;
  for (int left = steps; left > 0;) {
    int g = w.single ? 1 : group_length(left, steps);
    if (g > f.longest) g = f.longest;
    choose(l.gram_ts, [&](auto TS) {
      const Rider r = rides.next();
      const auto launch = [&](auto RIDE) {
        hipLaunchKernelGGL((ortho_gram_kernel<TS(), RIDE()>), dim3(r.blocks + l.n_gram), wg, 0, st, l, r, base, parts, w.kc, from);
      };
      if (r.blocks) launch(std::true_type());
      else launch(std::false_type());
      if (w.split) hipLaunchKernelGGL((ortho_sum_kernel<TS()>), dim3(l.n_gram, TS() / 32), wg, 0, st, l, base, parts);
    });
    const Stored R = brief ? brief_group(g) : group(g);
    left -= g;
    if (left) {
      choose(l.rect_ts, [&](auto TS) {
        const Rider r = rides.next();
        const auto launch = [&](auto RIDE) {
          hipLaunchKernelGGL((ortho_apply_kernel<TS(), RIDE()>), dim3(r.blocks + l.n_rect), wg, 0, st, l, r, base, parts, R.at,
                             1.f / R.scale, from);
        };
        if (r.blocks) launch(std::true_type());
        else launch(std::false_type());
      });
    } else {
      while (rides.left()) {
        const Rider r = rides.next();
        hipLaunchKernelGGL((ortho_square_kernel<Core64<8>, false, true>), dim3(r.blocks), dim3(512), 0, st, l, r, base, parts, Op{},
                           Op{});
      }
      choose(l.rect_ts, [&](auto TS) {
        const unsigned others = rides.c ? rides.c->n_rect : 0;
        hipLaunchKernelGGL((ortho_apply_last_kernel<T, TS()>), dim3(others + l.n_rect), wg, 0, st, lists.table, l,
                           Product{R.at, from, 1.f / R.scale}, second.rect, others, Product{SQ_F, rides.from, 1.f / SCALE}, base,
                           update, decay);
      });
    }
    from ^= 1;
    if (hipGetLastError() != hipSuccess) return -2;
  }
  return 0;
  };
  for (int k = 0; k < (riding ? 1 : p.chains); ++k) {
    const int rc = chain(lists.c[k], p.w[k]);
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace

size_t r3k_ortho_workspace_bytes(int count, const int* rows, const int* cols) {
  Plan p;
  return count > 0 && plan(count, rows, cols, p) == 0 ? p.total : 0;
}

int r3k_ortho(int count, const void* const* src, void* const* dst, float* const* buf, int dtype, const int* rows,
              const int* cols, const float* rates, float decay, float mu, int nesterov, int steps, float a, float b, float c,
              double eps, void* ws, size_t ws_bytes, hipStream_t st) {
  Plan p;
  if (plan(count, rows, cols, p) != 0 || dtype < 0 || dtype > 2 || steps < 1 || steps > 64 || !(eps >= 0)) return -1;
  const Poly f = polynomial(steps, a, b, c);
  if (!f.longest) return -1;
  if (count == 0) return 0;
  if (!src || !dst || (buf && !rates)) return -1;
  for (int i = 0; i < count; ++i)
    if (!src[i] || !dst[i] || (buf && !buf[i])) return -1;
  if (!ws || ws_bytes < p.total) return -3;
  char* w = static_cast<char*>(ws);
  if (reinterpret_cast<uintptr_t>(w) & 15) return -1;
  switch (dtype) {
    case 0: return run<float>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, f, eps, p, w, st);
    case 1: return run<_Float16>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, f, eps, p, w, st);
    default: return run<__bf16>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, f, eps, p, w, st);
  }
}
