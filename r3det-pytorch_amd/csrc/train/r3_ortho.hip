// r3_ortho.hip -- orthogonalising the updates of weight matrices by Newton-Schulz products, for a ragged list of matrices at
// once, alone or inside the optimiser's step (momentum before it, the weights' update behind it).
//
// For a matrix G (n x m, n <= m; a taller one is taken transposed):
//   X = G / (|G|_F + eps);   per step:  A = X X^t,  B = b A + c A A,  X <- a X + B X
// Each singular value s goes to a s + b s^3 + c s^5 while the singular vectors stay.  With the usual coefficients a small one
// grows by a = 3.44 a step, 485 in five, and so does every rounding of X: iterates rounded to 16 bits leave an error of
// 2-3 % in the result where the spectrum is a few directions over noise (fp16; 20 % in bf16).  So an iterate is held as
// TWO fp16 numbers, hi + lo, which together keep the 24 bits of fp32, and a product is three matrix products on the
// matrix cores, hi hi + hi lo + lo hi, summed in fp32 (lo lo is below fp32's own rounding).  Stored values carry a factor
// 2^12: |entries| <= the spectral norm <= 15 by the host's check of the coefficients, so hi does not overflow, and
// lo keeps its bits for entries down to 2^-12 of the largest.
//
// Every product has both operands with the summed index contiguous: X X^t and A A (A is symmetric) as they are, B X from
// X^t, which the kernel that makes X writes beside it.  X X^t and A A are symmetric: the tiles on and above the diagonal
// are computed, and written twice.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../r3_kernels.h"

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int TS = 64;           // tile of a product, and what matrices are padded to (with zeros, which stay zeros)
constexpr int BK = 32;           // of the summed index a stage holds
constexpr int NORM_CHUNK = 8192; // elements a workgroup of the norm's pass takes
constexpr float SCALE = 4096.f;  // what stored values are multiplied by
constexpr int WANT = 512;        // workgroups that fill the card

struct Mat {  // one matrix, as the device's table holds it
  const void* src;   // the matrix / the gradient
  void* dst;         // the result / the weights
  float* buf;        // the momentum (update only)
  int rows, cols;    // as the caller has it
  float rate;        // weights <- decay * weights - rate * result
  int splits;        // parts of the sum of X X^t
  unsigned tri0, rect0, norm0;  // first entries in the lists of triangle tiles (times splits), tiles, norm chunks
  unsigned part0;    // first partial tile
  size_t at;         // halves before this matrix's arrays
};
__host__ __device__ inline int up(int v) { return (v + TS - 1) / TS * TS; }
struct Dim {
  int n, m, np, mp, tn, tm;
  __host__ __device__ Dim(int rows, int cols) {
    n = rows < cols ? rows : cols;
    m = rows < cols ? cols : rows;
    np = up(n), mp = up(m), tn = np / TS, tm = mp / TS;
  }
  __host__ __device__ size_t x() const { return (size_t)np * mp; }
  __host__ __device__ size_t a() const { return (size_t)np * np; }
  // per matrix: X, X^t twice (read and written in the same pass), A, B; each hi then lo
  __host__ __device__ size_t halves() const { return 2 * (3 * x() + 2 * a()); }
  __host__ __device__ unsigned tri() const { return (unsigned)tn * (tn + 1) / 2; }
  __host__ __device__ unsigned rect() const { return (unsigned)tn * tm; }
  __host__ __device__ unsigned norms() const { return (unsigned)(((size_t)n * m + NORM_CHUNK - 1) / NORM_CHUNK); }
};
struct Area {  // where a matrix's arrays are
  _Float16 *x, *xt, *a, *b;  // xt: two of them
  __device__ Area(_Float16* base, const Mat& t, const Dim& d) {
    x = base + t.at;
    xt = x + 2 * d.x();
    a = xt + 4 * d.x();
    b = a + 2 * d.a();
  }
};
struct Tile {
  unsigned mat;
  unsigned short i, j;
  unsigned split;
};

// the whole workspace; every part is a multiple of 256 bytes
struct Plan {
  size_t table, tri, rect, norm_map, norms, counters, parts, halves, total;
  unsigned n_tri, n_rect, n_norm, n_part;
  int kc;  // the summed index of X X^t a workgroup takes at most
};

// ------------------------------------------------------------------------------------------------ the lists
constexpr int BATCH = 48;
struct Batch {
  Mat m[BATCH];
};
static_assert(sizeof(Batch) <= 3900, "a kernel's arguments hold 4 KB");
__global__ void ortho_table_kernel(Batch b, int count, Mat* table) {
  for (int i = threadIdx.x; i < count; i += blockDim.x) table[i] = b.m[i];
}

__device__ __forceinline__ unsigned find(const Mat* table, int count, unsigned Mat::* first, unsigned e) {
  int lo = 0, hi = count - 1;  // the last matrix that begins at or before e
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (table[mid].*first <= e) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
__global__ void ortho_lists_kernel(const Mat* table, int count, Tile* tri, unsigned n_tri, Tile* rect, unsigned n_rect,
                                   uint2* norm_map, unsigned n_norm, unsigned* counters, unsigned n_count) {
  const unsigned g = blockIdx.x * blockDim.x + threadIdx.x, stride = gridDim.x * blockDim.x;
  for (unsigned e = g; e < n_tri; e += stride) {
    const unsigned k = find(table, count, &Mat::tri0, e);
    const Mat& t = table[k];
    const Dim d(t.rows, t.cols);
    const unsigned local = e - t.tri0;
    unsigned tile = local / t.splits, i = 0;
    while (tile >= (unsigned)d.tn - i) tile -= d.tn - i, ++i;  // (row i has tn - i tiles)
    tri[e] = Tile{k, (unsigned short)i, (unsigned short)(i + tile), local % t.splits};
  }
  for (unsigned e = g; e < n_rect; e += stride) {
    const unsigned k = find(table, count, &Mat::rect0, e);
    const Dim d(table[k].rows, table[k].cols);
    const unsigned local = e - table[k].rect0;
    rect[e] = Tile{k, (unsigned short)(local % d.tn), (unsigned short)(local / d.tn), 0};
  }
  for (unsigned e = g; e < n_norm; e += stride) {
    const unsigned k = find(table, count, &Mat::norm0, e);
    norm_map[e] = make_uint2(k, e - table[k].norm0);
  }
  for (unsigned e = g; e < n_count; e += stride) counters[e] = 0;
}

// ------------------------------------------------------------------------------------------------ momentum, norm, X
template <typename T>
__device__ __forceinline__ float direction(const Mat& t, size_t i, bool update, float mu, bool nesterov) {
  const float g = (float)static_cast<const T*>(t.src)[i];
  if (!update) return g;
  return nesterov ? fmaf(mu, t.buf[i], g) : t.buf[i];
}
__device__ __forceinline__ double block_sum(double v, double* sh) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}
// momentum <- mu momentum + gradient, and the squares of the direction summed in 64 bits (no scaling of the matrix is needed
// against overflow, and the order of the sums is fixed)
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const Mat* __restrict__ table, const uint2* __restrict__ map,
                                                         double* __restrict__ norms, int update, float mu, int nesterov) {
  __shared__ double sh[4];
  const uint2 w = map[blockIdx.x];
  const Mat t = table[w.x];
  const size_t all = (size_t)t.rows * t.cols, from = (size_t)w.y * NORM_CHUNK;
  const size_t to = from + NORM_CHUNK < all ? from + NORM_CHUNK : all;
  double s = 0;
  for (size_t i = from + threadIdx.x; i < to; i += 256) {
    if (update) t.buf[i] = fmaf(mu, t.buf[i], (float)static_cast<const T*>(t.src)[i]);
    const double v = direction<T>(t, i, update, mu, nesterov);
    s = fma(v, v, s);
  }
  s = block_sum(s, sh);
  if (threadIdx.x == 0) norms[blockIdx.x] = s;
}

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}
// A tile of fp32 in shared memory, E[r][c] -> hi / lo arrays; rows of `ld`.
template <bool TURNED>
__device__ __forceinline__ void store_tile(const float (*E)[TS + 1], _Float16* p, size_t lo, size_t ld, int r0, int c0) {
#pragma unroll
  for (int q = threadIdx.x; q < TS * TS / 8; q += 256) {
    const int r = q / (TS / 8), c = q % (TS / 8) * 8;
    half8 h, l;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      _Float16 hh, ll;
      split16(TURNED ? E[c + k][r] : E[r][c + k], hh, ll);
      h[k] = hh, l[k] = ll;
    }
    _Float16* at = p + (size_t)(r0 + r) * ld + c0 + c;
    *reinterpret_cast<half8*>(at) = h;
    *reinterpret_cast<half8*>(at + lo) = l;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ortho_start_kernel(const Mat* __restrict__ table, const Tile* __restrict__ rect,
                                                          const double* __restrict__ norms, _Float16* __restrict__ base,
                                                          int update, float mu, int nesterov, double eps) {
  __shared__ double sh[4];
  __shared__ float E[TS][TS + 1];
  const Tile w = rect[blockIdx.x];
  const Mat t = table[w.mat];
  const Dim d(t.rows, t.cols);
  const Area o(base, t, d);
  double s = 0;
  for (unsigned i = threadIdx.x; i < d.norms(); i += 256) s += norms[t.norm0 + i];
  s = block_sum(s, sh);
  const double inv = (double)SCALE / (sqrt(s) + eps);
  const bool tall = t.rows > t.cols;
  const int i0 = w.i * TS, j0 = w.j * TS;
  for (int q = threadIdx.x; q < TS * TS; q += 256) {
    // (consecutive threads along the caller's rows)
    const int r = tall ? q % TS : q / TS, c = tall ? q / TS : q % TS;
    const int i = i0 + r, j = j0 + c;
    float v = 0.f;
    if (i < d.n && j < d.m) {
      const size_t at = tall ? (size_t)j * t.cols + i : (size_t)i * t.cols + j;
      v = (float)((double)direction<T>(t, at, update, mu, nesterov) * inv);
    }
    E[r][c] = v;
  }
  __syncthreads();
  store_tile<false>(E, o.x, d.x(), d.mp, i0, j0);
  store_tile<true>(E, o.xt, d.x(), d.np, j0, i0);
}

// ------------------------------------------------------------------------------------------------ the products
// One 64 x 64 tile of P Q^t by 4 wavefronts, 32 x 32 each: P, Q (hi, lo) with rows of ldp / ldq, the summed index
// [k0, k1).  A stage of 32 of it is 4 x 4 KB of shared memory, written by the loads themselves, two stages in turn.  A
// 16-byte piece c of row r sits at c ^ (r / 2 % 4): eight rows that are read together then lie in different banks.
struct Stage {
  half8 v[4][TS * BK / 8];
};
__device__ __forceinline__ void load_stage(Stage& s, const _Float16* p, size_t plo, size_t ldp, const _Float16* q, size_t qlo,
                                           size_t ldq, int k) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const _Float16* src = wave < 2 ? p + (wave & 1) * plo : q + (wave & 1) * qlo;
  const size_t ld = wave < 2 ? ldp : ldq;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int slot = t * 64 + lane, r = slot / 4, c = (slot % 4) ^ (r / 2 % 4);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + (size_t)r * ld + k + c * 8),
                                     (__attribute__((address_space(3))) void*)&s.v[wave][t * 64], 16, 0, 0);
  }
}
__device__ __forceinline__ void product(float16v& acc, Stage* st, const _Float16* p, size_t plo, size_t ldp, const _Float16* q,
                                        size_t qlo, size_t ldq, int k0, int k1) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int pr = (wave >> 1) * 32 + (lane & 31), qr = (wave & 1) * 32 + (lane & 31), kc = lane >> 5;
  load_stage(st[0], p, plo, ldp, q, qlo, ldq, k0);
  int cur = 0;
  for (int k = k0; k < k1; k += BK) {
    __syncthreads();  // this stage's loads are in, and everyone is done with the other stage
    if (k + BK < k1) load_stage(st[cur ^ 1], p, plo, ldp, q, qlo, ldq, k + BK);
    const Stage& s = st[cur];
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      const int ps = pr * 4 + ((kk * 2 + kc) ^ (pr / 2 % 4)), qs = qr * 4 + ((kk * 2 + kc) ^ (qr / 2 % 4));
      const half8 ph = s.v[0][ps], pl = s.v[1][ps], qh = s.v[2][qs], ql = s.v[3][qs];
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    }
    cur ^= 1;
  }
  __syncthreads();  // (the stages' memory is the epilogue's too)
}
union Shared {
  Stage st[2];
  float E[TS][TS + 1];
};
// lane l of the matrix instruction holds column l % 32 and rows 8 (r / 4) + 4 (l / 32) + r % 4
template <typename F>
__device__ __forceinline__ void each(const float16v& acc, const F& f) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    f((wave >> 1) * 32 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4, (wave & 1) * 32 + (lane & 31), acc[r]);
}

// A = X X^t: a tile on or above the diagonal, or one part of its sum.  The workgroup that ends a tile last adds the parts in
// their order, whoever it is, so results do not depend on the order of arrival.
__global__ __launch_bounds__(256) void ortho_gram_kernel(const Mat* __restrict__ table, const Tile* __restrict__ tri,
                                                         _Float16* base, float* parts, unsigned* counters, int kc) {
  __shared__ Shared sh;
  __shared__ unsigned last;
  const Tile w = tri[blockIdx.x];
  const Mat t = table[w.mat];
  const Dim d(t.rows, t.cols);
  const Area o(base, t, d);
  const int i0 = w.i * TS, j0 = w.j * TS;
  float16v acc = {};
  const int k0 = w.split * kc, k1 = k0 + kc < d.mp ? k0 + kc : d.mp;
  product(acc, sh.st, o.x + (size_t)i0 * d.mp, d.x(), d.mp, o.x + (size_t)j0 * d.mp, d.x(), d.mp, k0, k1);
  if (t.splits > 1) {
    const unsigned tile = (blockIdx.x - t.tri0) / t.splits;
    float* mine = parts + ((size_t)t.part0 + (size_t)tile * t.splits) * (TS * TS);
    each(acc, [&](int r, int c, float v) { mine[(size_t)w.split * (TS * TS) + r * TS + c] = v; });
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(&counters[t.part0 + tile], 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             (unsigned)t.splits - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    for (int q = threadIdx.x; q < TS * TS; q += 256) {
      float v = 0.f;
      for (int s = 0; s < t.splits; ++s) v += mine[(size_t)s * (TS * TS) + q];
      sh.E[q / TS][q % TS] = v * (1.f / SCALE);
    }
    if (threadIdx.x == 0) counters[t.part0 + tile] = 0;  // for the next step
  } else {
    each(acc, [&](int r, int c, float v) { sh.E[r][c] = v * (1.f / SCALE); });
  }
  __syncthreads();
  store_tile<false>(sh.E, o.a, d.a(), d.np, i0, j0);
  if (w.i != w.j) store_tile<true>(sh.E, o.a, d.a(), d.np, j0, i0);
}

// B = b A + c A A
__global__ __launch_bounds__(256) void ortho_poly_kernel(const Mat* __restrict__ table, const Tile* __restrict__ tri,
                                                         _Float16* base, float b, float c) {
  __shared__ Shared sh;
  const Tile w = tri[blockIdx.x];
  if (w.split) return;
  const Mat t = table[w.mat];
  const Dim d(t.rows, t.cols);
  const Area o(base, t, d);
  const int i0 = w.i * TS, j0 = w.j * TS;
  float16v acc = {};
  product(acc, sh.st, o.a + (size_t)i0 * d.np, d.a(), d.np, o.a + (size_t)j0 * d.np, d.a(), d.np, 0, d.np);
  each(acc, [&](int r, int q, float v) {
    const _Float16* p = o.a + (size_t)(i0 + r) * d.np + j0 + q;
    sh.E[r][q] = fmaf(b, (float)p[0] + (float)p[d.a()], c * (v * (1.f / SCALE)));
  });
  __syncthreads();
  store_tile<false>(sh.E, o.b, d.a(), d.np, i0, j0);
  if (w.i != w.j) store_tile<true>(sh.E, o.b, d.a(), d.np, j0, i0);
}

// X <- a X + B X, from X^t; the last step's goes to the caller, as the result or into the weights
template <typename T, bool LAST>
__global__ __launch_bounds__(256) void ortho_apply_kernel(const Mat* __restrict__ table, const Tile* __restrict__ rect,
                                                          _Float16* base, float a, int from, int update, float decay) {
  __shared__ Shared sh;
  const Tile w = rect[blockIdx.x];
  const Mat t = table[w.mat];
  const Dim d(t.rows, t.cols);
  const Area o(base, t, d);
  const int i0 = w.i * TS, j0 = w.j * TS;
  float16v acc = {};
  const _Float16* xt = o.xt + (from ? 2 * d.x() : 0);
  product(acc, sh.st, o.b + (size_t)i0 * d.np, d.a(), d.np, xt + (size_t)j0 * d.np, d.x(), d.np, 0, d.np);
  each(acc, [&](int r, int q, float v) {
    const _Float16* p = o.x + (size_t)(i0 + r) * d.mp + j0 + q;
    sh.E[r][q] = fmaf(a, (float)p[0] + (float)p[d.x()], v * (1.f / SCALE));
  });
  __syncthreads();
  if constexpr (!LAST) {
    store_tile<false>(sh.E, o.x, d.x(), d.mp, i0, j0);
    store_tile<true>(sh.E, o.xt + (from ? 0 : 2 * d.x()), d.x(), d.np, j0, i0);
  } else {
    const bool tall = t.rows > t.cols;
    T* out = static_cast<T*>(t.dst);
    for (int q = threadIdx.x; q < TS * TS; q += 256) {
      const int r = tall ? q % TS : q / TS, c = tall ? q / TS : q % TS;
      const int i = i0 + r, j = j0 + c;
      if (i < d.n && j < d.m) {
        const size_t at = tall ? (size_t)j * t.cols + i : (size_t)i * t.cols + j;
        const float v = sh.E[r][c] * (1.f / SCALE);
        out[at] = (T)(update ? fmaf(-t.rate, v, decay * (float)out[at]) : v);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ the host
size_t round256(size_t v) { return (v + 255) / 256 * 256; }

// 0: fine, -1: a shape that is not taken
int plan(int count, const int* rows, const int* cols, Plan& p) {
  if (count < 0 || count > (1 << 16) || (count && (!rows || !cols))) return -1;
  for (int i = 0; i < count; ++i) {
    if (rows[i] < 1 || cols[i] < 1 || (int64_t)rows[i] * cols[i] > 0x7fffffff) return -1;
    if ((rows[i] < cols[i] ? rows[i] : cols[i]) > 32768) return -1;
    if ((rows[i] > cols[i] ? rows[i] : cols[i]) > 65535 * TS) return -1;
  }
  // X X^t: the longest parts of the sum that still fill the card.  A part is a workgroup's time, so the parts of a ragged
  // list are of like length, and a short list of wide matrices is spread.
  for (p.kc = 4096; p.kc > 256; p.kc /= 2) {
    uint64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
      const Dim d(rows[i], cols[i]);
      blocks += (uint64_t)d.tri() * ((d.mp + p.kc - 1) / p.kc);
    }
    if (blocks >= WANT) break;
  }
  uint64_t tri = 0, rect = 0, norm = 0, part = 0, halves = 0;
  for (int i = 0; i < count; ++i) {
    const Dim d(rows[i], cols[i]);
    const unsigned s = (unsigned)((d.mp + p.kc - 1) / p.kc);
    tri += (uint64_t)d.tri() * s;
    rect += d.rect();
    norm += d.norms();
    part += (uint64_t)d.tri() * s;
    halves += d.halves();
  }
  if (tri > 0x7fffffff || rect > 0x7fffffff || norm > 0x7fffffff) return -1;
  p.n_tri = (unsigned)tri, p.n_rect = (unsigned)rect, p.n_norm = (unsigned)norm, p.n_part = (unsigned)part;
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t was = at;
    at += round256(bytes);
    return was;
  };
  p.table = take(sizeof(Mat) * (size_t)count);
  p.tri = take(sizeof(Tile) * tri);
  p.rect = take(sizeof(Tile) * rect);
  p.norm_map = take(sizeof(uint2) * norm);
  p.norms = take(sizeof(double) * norm);
  p.counters = take(sizeof(unsigned) * part);
  p.parts = take(sizeof(float) * TS * TS * part);
  p.halves = take(sizeof(_Float16) * halves);
  p.total = at;
  return 0;
}

// Whether every stored value stays below fp16's range: the spectral norms of X, A and B, from |X| <= 1 on, step by step, with
// the polynomial's extremes in between.  (1 % over, for the roundings of the iterates.)
bool bounded(int steps, double a, double b, double c) {
  if (!(fabs(a) < 1e6) || !(fabs(b) < 1e6) || !(fabs(c) < 1e6)) return false;
  const double most = 65504.0 / SCALE / 1.05;
  double top = 1;
  for (int k = 0; k < steps; ++k) {
    const auto X = [&](double s) { return fabs(s * (a + s * s * (b + s * s * c))); };
    const auto B = [&](double t) { return fabs(t * (b + t * c)); };
    const double t1 = top * top;
    double x = X(top), p = B(t1);
    const double tb = c != 0 ? -b / (2 * c) : -1;  // where b + 2 c t = 0
    if (tb > 0 && tb < t1) p = fmax(p, B(tb));
    // where a + 3 b t + 5 c t t = 0
    double t[2] = {-1, -1};
    if (c != 0) {
      const double q = 9 * b * b - 20 * a * c;
      if (q >= 0) t[0] = (-3 * b + sqrt(q)) / (10 * c), t[1] = (-3 * b - sqrt(q)) / (10 * c);
    } else if (b != 0) {
      t[0] = -a / (3 * b);
    }
    for (double v : t)
      if (v > 0 && v < t1) x = fmax(x, X(sqrt(v)));
    if (!(t1 <= most) || !(p <= most) || !(x <= most)) return false;
    top = 1.01 * x;
  }
  return true;
}

template <typename T>
int run(int count, const void* const* src, void* const* dst, float* const* buf, const int* rows, const int* cols,
        const float* rates, float decay, float mu, int nesterov, int steps, float a, float b, float c, double eps,
        const Plan& p, char* ws, hipStream_t st) {
  Mat* table = reinterpret_cast<Mat*>(ws + p.table);
  Tile* tri = reinterpret_cast<Tile*>(ws + p.tri);
  Tile* rect = reinterpret_cast<Tile*>(ws + p.rect);
  uint2* norm_map = reinterpret_cast<uint2*>(ws + p.norm_map);
  double* norms = reinterpret_cast<double*>(ws + p.norms);
  unsigned* counters = reinterpret_cast<unsigned*>(ws + p.counters);
  float* parts = reinterpret_cast<float*>(ws + p.parts);
  _Float16* base = reinterpret_cast<_Float16*>(ws + p.halves);
  const int update = buf != nullptr;
  unsigned n_tri = 0, n_rect = 0, n_norm = 0;
  size_t halves = 0;
  for (int first = 0; first < count; first += BATCH) {
    Batch batch;
    const int many = count - first < BATCH ? count - first : BATCH;
    for (int k = 0; k < many; ++k) {
      const int i = first + k;
      const Dim d(rows[i], cols[i]);
      const unsigned s = (unsigned)((d.mp + p.kc - 1) / p.kc);
      batch.m[k] = Mat{src[i], dst[i], update ? buf[i] : nullptr, rows[i], cols[i], rates ? rates[i] : 0.f, (int)s, n_tri,
                       n_rect, n_norm, n_tri, halves};
      n_tri += d.tri() * s;
      n_rect += d.rect();
      n_norm += d.norms();
      halves += d.halves();
    }
    hipLaunchKernelGGL(ortho_table_kernel, dim3(1), dim3(64), 0, st, batch, many, table + first);
    if (hipGetLastError() != hipSuccess) return -2;
  }
  unsigned blocks = (n_rect > n_tri ? n_rect : n_tri) / 256 + 1;
  if (blocks > 1024) blocks = 1024;
  hipLaunchKernelGGL(ortho_lists_kernel, dim3(blocks), dim3(256), 0, st, table, count, tri, n_tri, rect, n_rect, norm_map,
                     n_norm, counters, p.n_part);
  hipLaunchKernelGGL((ortho_norm_kernel<T>), dim3(n_norm), dim3(256), 0, st, table, norm_map, norms, update, mu, nesterov);
  hipLaunchKernelGGL((ortho_start_kernel<T>), dim3(n_rect), dim3(256), 0, st, table, rect, norms, base, update, mu, nesterov, eps);
  if (hipGetLastError() != hipSuccess) return -2;
  for (int k = 0; k < steps; ++k) {
    hipLaunchKernelGGL(ortho_gram_kernel, dim3(n_tri), dim3(256), 0, st, table, tri, base, parts, counters, p.kc);
    hipLaunchKernelGGL(ortho_poly_kernel, dim3(n_tri), dim3(256), 0, st, table, tri, base, b, c);
    if (k + 1 < steps)
      hipLaunchKernelGGL((ortho_apply_kernel<T, false>), dim3(n_rect), dim3(256), 0, st, table, rect, base, a, k & 1, update,
                         decay);
    else
      hipLaunchKernelGGL((ortho_apply_kernel<T, true>), dim3(n_rect), dim3(256), 0, st, table, rect, base, a, k & 1, update,
                         decay);
    if (hipGetLastError() != hipSuccess) return -2;
  }
  return 0;
}

}  // namespace

size_t r3k_ortho_workspace_bytes(int count, const int* rows, const int* cols) {
  Plan p;
  return plan(count, rows, cols, p) == 0 ? p.total : 0;
}

int r3k_ortho(int count, const void* const* src, void* const* dst, float* const* buf, int dtype, const int* rows,
              const int* cols, const float* rates, float decay, float mu, int nesterov, int steps, float a, float b, float c,
              double eps, void* ws, size_t ws_bytes, hipStream_t st) {
  Plan p;
  if (plan(count, rows, cols, p) != 0 || dtype < 0 || dtype > 2 || steps < 1 || steps > 64 || !(eps >= 0) ||
      !bounded(steps, a, b, c))
    return -1;
  if (count == 0) return 0;
  if (!src || !dst || (buf && !rates)) return -1;
  for (int i = 0; i < count; ++i)
    if (!src[i] || !dst[i] || (buf && !buf[i])) return -1;
  if (!ws || ws_bytes < p.total) return -3;
  char* w = static_cast<char*>(ws);
  if (reinterpret_cast<uintptr_t>(w) & 15) return -1;
  switch (dtype) {
    case 0: return run<float>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, a, b, c, eps, p, w, st);
    case 1: return run<_Float16>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, a, b, c, eps, p, w, st);
    default: return run<__bf16>(count, src, dst, buf, rows, cols, rates, decay, mu, nesterov, steps, a, b, c, eps, p, w, st);
  }
}
