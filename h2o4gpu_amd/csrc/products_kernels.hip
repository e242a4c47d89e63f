// Products grouped by expert: rows in expert order times each expert's matrix, and the two gradients.
//
//   product:          y[p] = W[e] x[p]                     p in [offsets[e], offsets[e + 1])
//   product_drows:    dx[p] = W[e]^T dy[p]
//   product_dweights: dW[e] = sum over p of dy[p] x[p]^T
//
// Sums are float32, in an order that depends on the sizes and the offsets alone; one rounding at the end. Long products
// of rows that begin at words go to pipe_kernel, those of few rows to thin_kernel, and what is left is here.
#include "product_thin.h"

namespace kmhip {
namespace {

struct ProductArgs {
  const void *x;  // m's operand: rows in expert order (dy of DWEIGHTS)
  const void *w;  // n's operand: the matrices (x of DWEIGHTS)
  void *c;
  size_t x_stride, w_stride, w_expert, c_stride, c_expert;
  const int *offsets;
  int experts, rows, n, k;  // DWEIGHTS: n = cols, k = out, which is C's m
  int part;                 // DWEIGHTS: rows of a part
  float *sums;              // of experts with several: matrices like C's, float
  unsigned first_block;
  int n_tiles;
};

// Any alignment and any sizes: pieces come through registers, masked at the edges, the next stage's while this one is
// multiplied. A wavefront's shifts and masks take about as long as its products, so a CU has three workgroups of 2-byte
// elements, with one buffer of LDS each: 28800 rows of 300 experts of 777 x 1001 take 195 us, with two buffers, two
// workgroups, 205 (their matrices' gradient 304 and 339); 4096 rows of 8 experts of 2049 x 4047 214 and 242. Of float32,
// which the matrix instructions bound, it is two: 64000 rows of 16 experts of 96 x 1024 118 us, with one buffer 127 (145 and
// 180). HALVES: some row of an operand of 2-byte elements begins between two words.
template <typename T, Kind KIND, bool HALVES, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, sizeof(T) == 4 ? 2 : 3) void product_kernel(ProductArgs a) {
  constexpr bool XC = KIND == DWEIGHTS, WC = KIND != FORWARD;
  typedef OperandTile<T, BM, XC> TX;
  typedef OperandTile<T, BN, WC> TW;
  constexpr int THREADS = WM * WN * 64, KS = TX::KS, EPP = TX::EPP;
  constexpr int PX = TX::SLOTS / THREADS, PW = TW::SLOTS / THREADS;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int STAGE = (BM + BN) * 128, BUFFERS = sizeof(T) == 4 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) char lds[BUFFERS * STAGE];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned block = a.first_block + blockIdx.x, number = block / (unsigned)a.n_tiles;
  const int n0 = (int)(block % (unsigned)a.n_tiles) * BN;
  int expert, first, m_here;
  const T *x = static_cast<const T *>(a.x), *w = static_cast<const T *>(a.w);
  T *c = static_cast<T *>(a.c);
  int k_end = a.k;
  float *sum = nullptr;  // C is a part's sum
  if (KIND == DWEIGHTS) {
    const int tiles = (a.k + BM - 1) / BM;
    PartOfRows part;
    if (!part_of_rows(a.offsets, a.experts, a.rows, a.part, number / tiles, part)) return;
    expert = part.expert, k_end = part.rows;
    first = (number % tiles) * BM;
    m_here = a.k - first < BM ? a.k - first : BM;
    x += (size_t)part.first * a.x_stride + first;
    w += (size_t)part.first * a.w_stride;
    c += (size_t)expert * a.c_expert + (size_t)first * a.c_stride;
    if (part.sum >= 0) sum = a.sums + (size_t)part.sum * a.c_expert + (size_t)first * a.c_stride;
  } else {
    if (!ragged_tile(a.offsets, a.experts, a.rows, BM, number, expert, first, m_here)) return;
    x += (size_t)first * a.x_stride;
    c += (size_t)first * a.c_stride;
    w += (size_t)expert * a.w_expert;
    if (expert == a.experts) k_end = 0;  // rows without an expert: zeros
  }
  const int n_here = a.n - n0 < BN ? a.n - n0 : BN;
  w += WC ? (size_t)n0 : (size_t)n0 * a.w_stride;

  // A stage of an operand: its first word, its size up to the last word that holds any of it, and what its first element
  // lies behind the first word. What is behind the end is not read. Behind the last k may lie anything (the next row, or
  // the half of the last word that is not the operand's): settle() takes it out; of rows and columns that do not exist
  // nothing is stored.
  struct Stage {
    const char *from;
    unsigned size, behind;
  };
  auto stage_of = [&](const T *first_element, size_t lines, size_t stride, size_t side) {
    const size_t at = (size_t)first_element;
    const unsigned behind = (unsigned)(at & 3);
    const unsigned size = lines > 0 && side > 0 ? (unsigned)(((lines - 1) * stride + side) * sizeof(T)) + behind : 0;
    return Stage{(const char *)(at - behind), (size + 3) & ~3u, behind};
  };
  const auto stage_x = [&](int k0) {
    const int left = k_end - k0;
    return XC ? stage_of(x + (size_t)k0 * a.x_stride, left < KS ? left : KS, a.x_stride, m_here)
              : stage_of(x + k0, m_here, a.x_stride, left);
  };
  const auto stage_w = [&](int k0) {
    const int left = k_end - k0;
    return WC ? stage_of(w + (size_t)k0 * a.w_stride, left < KS ? left : KS, a.w_stride, n_here)
              : stage_of(w + k0, n_here, a.w_stride, left);
  };
  u32x4 px[PX], pw[PW];
  unsigned last_x[HALVES ? PX : 1], last_w[HALVES ? PW : 1];
  auto load = [&](int k0) __attribute__((always_inline)) {
    const Stage sx = stage_x(k0), sw = stage_w(k0);
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      int r, k;
      TX::place(i * THREADS + tid, r, k);
      const unsigned at = (unsigned)((XC ? k * a.x_stride + r : r * a.x_stride + k) * sizeof(T)) + sx.behind;
      px[i] = buffer_words(sx.from, sx.size, HALVES ? at & ~3u : at);
      if (HALVES) last_x[i] = buffer_word(sx.from, sx.size, (at + 14) & ~3u);
    }
#pragma unroll
    for (int i = 0; i < PW; ++i) {
      int r, k;
      TW::place(i * THREADS + tid, r, k);
      const unsigned at = (unsigned)((WC ? k * a.w_stride + r : r * a.w_stride + k) * sizeof(T)) + sw.behind;
      pw[i] = buffer_words(sw.from, sw.size, HALVES ? at & ~3u : at);
      if (HALVES) last_w[i] = buffer_word(sw.from, sw.size, (at + 14) & ~3u);
    }
  };
  // 2-byte elements that lie between words are shifted, and behind the last k are zeros
  auto settle = [&](int k0) __attribute__((always_inline)) {
    if constexpr (HALVES) {
      const unsigned bx = stage_x(k0).behind, bw = stage_w(k0).behind;
#pragma unroll
      for (int i = 0; i < PX; ++i) {
        int r, k;
        TX::place(i * THREADS + tid, r, k);
        px[i] = shifted(px[i], last_x[i], (bx + (unsigned)((XC ? k * a.x_stride + r : r * a.x_stride + k) * 2)) & 2);
      }
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        int r, k;
        TW::place(i * THREADS + tid, r, k);
        pw[i] = shifted(pw[i], last_w[i], (bw + (unsigned)((WC ? k * a.w_stride + r : r * a.w_stride + k) * 2)) & 2);
      }
    }
    if (k0 + KS > k_end) {
#pragma unroll
      for (int i = 0; i < PX; ++i) {
        int r, k;
        TX::place(i * THREADS + tid, r, k);
        px[i] &= first_of<T>(XC ? (k < k_end - k0 ? EPP : 0) : k_end - k0 - k);
      }
#pragma unroll
      for (int i = 0; i < PW; ++i) {
        int r, k;
        TW::place(i * THREADS + tid, r, k);
        pw[i] &= first_of<T>(WC ? (k < k_end - k0 ? EPP : 0) : k_end - k0 - k);
      }
    }
  };
  auto put = [&](char *at) {
#pragma unroll
    for (int i = 0; i < PX; ++i) *reinterpret_cast<u32x4 *>(at + (i * THREADS + tid) * 16) = px[i];
#pragma unroll
    for (int i = 0; i < PW; ++i) *reinterpret_cast<u32x4 *>(at + BM * 128 + (i * THREADS + tid) * 16) = pw[i];
  };

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // blocks of 16 go round the wavefronts, so that they have as many each where a tile is not full
  const int wm = wave / WN, wn = wave % WN;
  const int m_blocks = ((m_here + 15) / 16 - wm + WM - 1) / WM, n_blocks = ((n_here + 15) / 16 - wn + WN - 1) / WN;
  const int stages = (k_end + KS - 1) / KS;
  if (stages > 0) {
    load(0);
    settle(0);
    put(lds);
  }
  __syncthreads();
  for (int t = 0; t < stages; ++t) {
    const char *at = lds + (BUFFERS == 2 ? (t & 1) * STAGE : 0);
    if (t + 1 < stages) load((t + 1) * KS);
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      if (step == 1 && k_end - t * KS <= KS / 2) break;  // (zeros)
      u32x4 fx[FM], fw[FN];
#pragma unroll
      for (int i = 0; i < FM; ++i) fx[i] = TX::fragment(at, lane, i * WM + wm, step);
#pragma unroll
      for (int j = 0; j < FN; ++j) fw[j] = TW::fragment(at + BM * 128, lane, j * WN + wn, step);
#pragma unroll
      for (int i = 0; i < FM; ++i)
        if (i < m_blocks) {
#pragma unroll
          for (int j = 0; j < FN; ++j)
            if (j < n_blocks) mfma_piece(acc[i][j], fw[j], fx[i], Tag<T>());
        }
    }
    if (BUFFERS == 1) __syncthreads();
    if (t + 1 < stages) {
      settle((t + 1) * KS);
      put(lds + (BUFFERS == 2 ? ((t + 1) & 1) * STAGE : 0));
    }
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = (i * WM + wm) * 16 + (lane & 15);
    if (m >= m_here) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = (j * WN + wn) * 16 + 4 * (lane >> 4);
      if (KIND == DWEIGHTS && sum)
        store_four(sum + (size_t)m * a.c_stride + n0 + n, acc[i][j], n_here - n);
      else
        store_four(c + (size_t)m * a.c_stride + n0 + n, acc[i][j], n_here - n);
    }
  }
}

// The parts' sums of the experts that have several, added up in order: a workgroup has a stretch of the matrix of the
// expert whose first part begins in its `part` rows, a thread an element. What the parts' sums take to be read bounds it (98
// parts of 2 experts of 101 x 101: 6 us).
template <typename T>
__global__ __launch_bounds__(256) void join_parts_kernel(const float *sums, const int *offsets, int experts, int part,
                                                         size_t size, T *c) {
  const int window = blockIdx.y;
  const long long end = (long long)(window + 1) * part;  // the last expert that begins within or before these rows
  const int lo = last_below(offsets, experts, end < INT_MAX ? (int)end - 1 : INT_MAX);
  const int begin = offsets[lo], rows = offsets[lo + 1] - begin;
  if (begin / part != window || rows <= part) return;
  const size_t at = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= size) return;
  const int parts = (rows + part - 1) / part;
  const float *from = sums + (size_t)(2 * window + 1) * size + at;  // of the first part; then every second
  float total = *from;
  from += size;
  for (int j = 1; j < parts; j += 8) {  // (eight loads on their way at once)
    float next[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) next[i] = j + i < parts ? from[(size_t)2 * (j + i - 1) * size] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < parts) total += next[i];
  }
  c[(size_t)lo * size + at] = (T)total;
}

// Whether every row of both operands begins at a multiple of 16 bytes.
template <typename T>
bool rows_aligned(const ProductArgs &a) {
  constexpr size_t EPP = 16 / sizeof(T);
  return aligned_to(a.x, 16) && aligned_to(a.w, 16) && a.x_stride % EPP == 0 && a.w_stride % EPP == 0 &&
         (a.experts == 1 || a.w_expert % EPP == 0);
}

template <typename T>
int join_parts(const ProductArgs &a, hipStream_t stream) {
  if (a.rows <= a.part) return H2O4GPU_KMEANS_OK;
  const size_t blocks = (a.c_expert + 255) / 256;
  hipLaunchKernelGGL((join_parts_kernel<T>), dim3((unsigned)blocks, (unsigned)(a.rows / a.part + 1)), dim3(256), 0, stream,
                     a.sums, a.offsets, a.experts, a.part, a.c_expert, static_cast<T *>(a.c));
  return launched();
}

template <typename T, Kind KIND>
int launch_product(const ProductArgs &a, hipStream_t stream) {
  const ProductSizes sizes = {KIND,       (int)sizeof(T), a.x, a.w, a.x_stride, a.w_stride, a.w_expert, a.experts,
                              a.rows, a.n,            a.k, a.part};
  const bool halves = between_words(sizes);
  const Way way = way_of(sizes);
  if (KIND != DWEIGHTS && way == FEW_ROWS) {
    ThinArgs t = {};
    t.x = static_cast<const char *>(a.x), t.w = static_cast<const char *>(a.w), t.c = a.c;
    t.x_stride = a.x_stride * sizeof(T), t.w_stride = a.w_stride * sizeof(T), t.w_expert = a.w_expert * sizeof(T);
    t.c_stride = a.c_stride, t.offsets = a.offsets;
    t.experts = a.experts, t.rows = a.rows, t.n = a.n, t.k = a.k;
    t.halves = halves;
    if (KIND == DROWS) return launch_thin_columns<T>(t, stream);
    return rows_aligned<T>(a) && a.k % (16 / sizeof(T)) == 0 ? launch_thin<T, T, true>(t, stream)
                                                             : launch_thin<T, T, false>(t, stream);
  }
  if (way == TILES_128 || way == TILES_256) {
    PipeArgs p = {};
    p.x = static_cast<const char *>(a.x), p.w = static_cast<const char *>(a.w), p.c = a.c;
    p.x_stride = a.x_stride * sizeof(T), p.w_stride = a.w_stride * sizeof(T), p.w_expert = a.w_expert * sizeof(T);
    p.c_stride = a.c_stride, p.c_expert = a.c_expert;
    p.offsets = a.offsets, p.experts = a.experts, p.rows = a.rows, p.n = a.n, p.k = a.k;
    p.part = a.part, p.sums = a.sums;
    KM_TRY((launch_large<T, T, KIND, false>(p, way, stream)));
    return KIND == DWEIGHTS ? join_parts<T>(a, stream) : H2O4GPU_KMEANS_OK;
  }
  constexpr int BM = 128, BN = 128;
  const size_t m_tiles = KIND == DWEIGHTS ? ragged_tiles(a.experts, a.rows, a.part) * ((a.k + BM - 1) / BM)
                                          : ragged_tiles(a.experts, a.rows, BM);
  ProductArgs p = a;
  p.n_tiles = (a.n + BN - 1) / BN;
  KM_TRY(in_launches(m_tiles * p.n_tiles, [&](unsigned first, unsigned blocks) {
    p.first_block = first;
    if (sizeof(T) == 2 && halves)
      hipLaunchKernelGGL((product_kernel<T, KIND, sizeof(T) == 2, BM, BN, 2, 2>), dim3(blocks), dim3(256), 0, stream, p);
    else
      hipLaunchKernelGGL((product_kernel<T, KIND, false, BM, BN, 2, 2>), dim3(blocks), dim3(256), 0, stream, p);
    return launched();
  }));
  return KIND == DWEIGHTS ? join_parts<T>(a, stream) : H2O4GPU_KMEANS_OK;
}

// Where elements of a type may lie.
bool elements(int dtype, const void *p) { return p && aligned_to(p, type_size(dtype)); }

// Strides of rows of `cols` elements, each row apart from the next.
bool fits(size_t rows, size_t cols, size_t stride) { return rows < 2 || stride >= cols; }

// A thread a piece of 16 bytes: rows as they come, into rows that begin at multiples of 16 bytes, zeros behind their ends.
// Bound by memory: 456750 rows of 781 (bfloat16, 714 MB in, 716 out) take 355 us, 4.0 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void align_kernel(const T *in, size_t stride, size_t matrix, size_t rows, size_t cols,
                                                    size_t pieces, size_t total, u32x4 *out, unsigned first_block) {
  const size_t at = (size_t)(first_block + blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const size_t row = at / pieces, col = (at - row * pieces) * (16 / sizeof(T)), of = row / rows;
  const size_t left = cols - col;
  out[at] = load_piece(in + of * matrix + (row - of * rows) * stride + col, left < 16 ? (int)left : 16);
}

constexpr size_t MAX_SIDE = (size_t)1 << 30;

// What all three have in common. > 0: go on, else the status to return.
int check(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *offsets, size_t w_stride = 0) {
  if (!known_type(dtype) || experts < 1 || experts > H2O4GPU_EXPERTS_MAX_EXPERTS) return H2O4GPU_KMEANS_EARG;
  if (out < 1 || cols < 1 || out > MAX_SIDE || cols > MAX_SIDE || rows > (size_t)INT_MAX - 65536 || !offsets ||
      (out > 1 && w_stride > ((size_t)1 << 23)))  // (64 rows of a matrix are within a buffer's reach)
    return H2O4GPU_KMEANS_EARG;
  return 1;
}

}  // namespace
}  // namespace kmhip

using namespace kmhip;

KM_API int h2o4gpu_experts_product(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *d_rows,
                                   size_t rows_stride, const void *d_weights, size_t expert_stride, size_t w_stride,
                                   const int *d_offsets, void *d_y, size_t y_stride, void *stream) {
  if (int rc = check(dtype, rows, experts, out, cols, rows ? (const void *)d_offsets : "", w_stride);
      rc <= 0)
    return rc;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!elements(dtype, d_rows) || !elements(dtype, d_weights) || !elements(dtype, d_y))
    return H2O4GPU_KMEANS_EARG;
  if (!fits(rows, cols, rows_stride) || !fits(out, cols, w_stride) ||
      !fits(rows, out, y_stride))
    return H2O4GPU_KMEANS_EARG;
  ProductArgs a = {d_rows, d_weights, d_y, rows_stride, w_stride, expert_stride, y_stride, 0, d_offsets, experts, (int)rows,
                   (int)out, (int)cols, 0, nullptr, 0, 0};
  return with_type(dtype, [&](auto tag) {
    return launch_product<typename decltype(tag)::type, FORWARD>(a, static_cast<hipStream_t>(stream));
  });
}

KM_API int h2o4gpu_experts_product_drows(int dtype, size_t rows, int experts, size_t out, size_t cols, const void *d_dy,
                                         size_t dy_stride, const void *d_weights, size_t expert_stride, size_t w_stride,
                                         const int *d_offsets, void *d_drows, size_t drows_stride, void *stream) {
  if (int rc = check(dtype, rows, experts, out, cols, rows ? (const void *)d_offsets : "", w_stride); rc <= 0)
    return rc;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!elements(dtype, d_dy) || !elements(dtype, d_weights) || !elements(dtype, d_drows))
    return H2O4GPU_KMEANS_EARG;
  if (!fits(rows, out, dy_stride) || !fits(out, cols, w_stride) ||
      !fits(rows, cols, drows_stride))
    return H2O4GPU_KMEANS_EARG;
  ProductArgs a = {d_dy, d_weights, d_drows, dy_stride, w_stride, expert_stride, drows_stride, 0, d_offsets, experts,
                   (int)rows, (int)cols, (int)out, 0, nullptr, 0, 0};
  return with_type(dtype, [&](auto tag) {
    return launch_product<typename decltype(tag)::type, DROWS>(a, static_cast<hipStream_t>(stream));
  });
}

KM_API size_t h2o4gpu_experts_product_dweights_workspace(int dtype, size_t rows, int experts, size_t out, size_t cols) {
  return check(dtype, rows, experts, out, cols, "") <= 0 ? 0 : sums_bytes(type_size(dtype), rows, experts, out, cols);
}

KM_API int h2o4gpu_experts_product_dweights(int dtype, size_t rows, int experts, size_t out, size_t cols,
                                            const void *d_dy, size_t dy_stride, const void *d_rows, size_t rows_stride,
                                            const int *d_offsets, void *d_dweights, void *d_workspace,
                                            size_t workspace_bytes, void *stream) {
  if (int rc = check(dtype, rows, experts, out, cols, d_offsets); rc <= 0) return rc;
  const size_t need = sums_bytes(type_size(dtype), rows, experts, out, cols);
  if (need > workspace_bytes || (need && (!d_workspace || !aligned_to(d_workspace, 16)))) return H2O4GPU_KMEANS_EARG;
  if (out > H2O4GPU_EXPERTS_MAX_SIDE || cols > H2O4GPU_EXPERTS_MAX_SIDE ||
      (rows > 1 && (dy_stride > H2O4GPU_EXPERTS_MAX_SIDE || rows_stride > H2O4GPU_EXPERTS_MAX_SIDE)))
    return H2O4GPU_KMEANS_EARG;
  if (!elements(dtype, d_dweights) || (rows && (!elements(dtype, d_dy) || !elements(dtype, d_rows))))
    return H2O4GPU_KMEANS_EARG;
  if (!fits(rows, out, dy_stride) || !fits(rows, cols, rows_stride))
    return H2O4GPU_KMEANS_EARG;
  ProductArgs a = {d_dy, d_rows, d_dweights, dy_stride, rows_stride, 0, cols, out * cols, d_offsets, experts, (int)rows,
                   (int)cols, (int)out, 0, nullptr, 0, 0};
  a.part = rows_of_part(type_size(dtype), rows, experts, out, cols), a.sums = static_cast<float *>(d_workspace);
  return with_type(dtype, [&](auto tag) {
    return launch_product<typename decltype(tag)::type, DWEIGHTS>(a, static_cast<hipStream_t>(stream));
  });
}

KM_API int h2o4gpu_experts_align_rows(int dtype, size_t matrices, size_t rows, size_t cols, const void *d_in,
                                      size_t matrix_stride, size_t stride, void *d_out, void *stream) {
  if (!known_type(dtype) || cols < 1 || cols > MAX_SIDE || rows > (size_t)INT_MAX || matrices > (size_t)INT_MAX)
    return H2O4GPU_KMEANS_EARG;
  const size_t size = type_size(dtype), pieces = (cols * size + 15) / 16;
  if (matrices * rows > ((size_t)1 << 40) / pieces) return H2O4GPU_KMEANS_EARG;
  const size_t total = matrices * rows * pieces;
  if (total == 0) return H2O4GPU_KMEANS_OK;
  if (!elements(dtype, d_in) || !d_out || !aligned_to(d_out, 16)) return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    return in_launches((total + 255) / 256, [&](unsigned first, unsigned here) {
      hipLaunchKernelGGL((align_kernel<T>), dim3(here), dim3(256), 0, static_cast<hipStream_t>(stream),
                         static_cast<const T *>(d_in), stride, matrix_stride, rows, cols, pieces, total,
                         static_cast<u32x4 *>(d_out), first);
      return launched();
    });
  });
}
