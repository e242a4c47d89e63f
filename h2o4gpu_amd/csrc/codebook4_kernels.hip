// Matrices of 4-bit codes: compressing one, and its product with tokens, alone or a matrix per expert.
#include "experts_common.h"

namespace kmhip {

// ---------------------------------------------------------------------------
// compressing
// ---------------------------------------------------------------------------

// One wavefront a row, a group at a time: largest magnitude, scale, then the nearest entry of every
// element, two to a byte. (Weights are compressed once: nothing here is made fast.)
template <typename T, typename S>
__global__ __launch_bounds__(256) void quantize4_kernel(const T *w, int64_t ws, int64_t out, int cols, int group,
                                                        float top, const T *book, uint8_t *codes, int64_t pitch,
                                                        S *scales) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= out) return;
  const int groups = (cols + group - 1) / group;
  for (int g = 0; g < groups; g++) {
    const int lo = g * group, hi = lo + group < cols ? lo + group : cols;
    float most = 0.f;
    for (int k = lo + lane; k < hi; k += 64) most = fmaxf(most, fabsf((float)w[n * ws + k]));
    for (int m = 32; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor(most, m, 64));
    S scale = (S)(most / top);
    if (!((float)scale > 0.f) || !isfinite((float)scale)) scale = (S)1.f;
    if (lane == 0) scales[n * groups + g] = scale;
    const float by = (float)scale;
    for (int b = lo / 2 + lane; b < (hi + 1) / 2; b += 64) {
      unsigned byte = 0;
      for (int h = 0; h < 2; h++) {
        const int k = 2 * b + h;
        if (k >= hi) continue;
        const float v = (float)w[n * ws + k] / by;
        float best = __builtin_huge_valf();
        unsigned code = 0;
        for (int c = 0; c < 16; c++) {
          const float off = fabsf(v - (float)book[c]);
          if (off < best) {
            best = off;
            code = c;
          }
        }
        byte |= code << (4 * h);
      }
      codes[n * pitch + b] = (uint8_t)byte;
    }
  }
  for (int64_t b = (cols + 1) / 2 + lane; b < pitch; b += 64) codes[n * pitch + b] = 0;
}

// ---------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------

// Which rows a launch has: all of x against one matrix (offsets == nullptr), or every expert's.
struct RowSource {
  const int *order = nullptr, *offsets = nullptr;
  int top_k = 1, experts = 1;
  int64_t rows = 0;  // of y
};

struct Matrix4 {
  const uint8_t *codes = nullptr;
  int64_t pitch = 0, out = 0;
  int cols = 0, group = 0, groups = 0;
  int64_t book_stride = 0;
};

// One wavefront a column of y and four rows of it at a time; blockIdx.y is the expert, the last one
// writes the zeros of the rows that have none.
template <typename T, typename S>
__global__ __launch_bounds__(256) void product4_any_kernel(const T *x, int64_t xs, Matrix4 m, const S *scales,
                                                           const T *books, RowSource src, T *y, int64_t ys) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int e = blockIdx.y;
  __shared__ float book[16];
  int64_t lo = 0, hi = src.rows;
  if (src.offsets) {
    lo = src.offsets[e];
    if (e < src.experts) hi = src.offsets[e + 1];
  }
  if (lo >= hi) return;
  if (src.offsets && e == src.experts) {
    if (n < m.out)
      for (int64_t p = lo + lane; p < hi; p += 64) y[p * ys + n] = (T)0.f;
    return;
  }
  if (threadIdx.x < 16) book[threadIdx.x] = (float)books[e * m.book_stride + threadIdx.x];
  __syncthreads();
  if (n >= m.out) return;
  const uint8_t *codes = m.codes + ((int64_t)e * m.out + n) * m.pitch;
  const S *sc = scales + ((int64_t)e * m.out + n) * m.groups;
  for (int64_t p = lo; p < hi; p += 4) {
    float acc[4] = {};
    const T *xp[4];
    for (int r = 0; r < 4; r++) {
      const int64_t q = p + r < hi ? p + r : hi - 1;
      xp[r] = x + (src.order ? src.order[q] / src.top_k : q) * xs;
    }
    for (int k = 8 * lane; k < m.cols; k += 512) {
      const unsigned word = *reinterpret_cast<const unsigned *>(codes + k / 2);
      const float scale = (float)sc[k / m.group];
      for (int i = 0; i < 8; i++) {
        if (k + i >= m.cols) break;
        const float v = book[(word >> (4 * i)) & 15] * scale;
        for (int r = 0; r < 4; r++) acc[r] = fmaf(v, (float)xp[r][k + i], acc[r]);
      }
    }
    for (int r = 0; r < 4; r++) {
      for (int o = 32; o >= 1; o >>= 1) acc[r] += __shfl_xor(acc[r], o, 64);
      if (lane == 0 && p + r < hi) y[(p + r) * ys + n] = (T)acc[r];
    }
  }
}

static const size_t MOST_OUT = 1 << 24, MOST_COLS4 = 1000000, MOST_ROWS4 = 2147483646;

static bool matrix_ok(int dtype, size_t out, size_t cols, int group, const void *codes, size_t pitch, int scale_dtype,
                      const void *scales, const void *book) {
  return known_type(dtype) && known_type(scale_dtype) && out >= 1 && out <= MOST_OUT && cols >= 1 &&
         cols <= MOST_COLS4 && group >= 32 && group % 32 == 0 && codes && aligned_to(codes, 16) && pitch % 16 == 0 &&
         pitch >= (cols + 1) / 2 && pitch <= ((size_t)1 << 32) && scales &&
         aligned_to(scales, type_size(scale_dtype)) && book && aligned_to(book, type_size(dtype));
}

static bool strided_ok(int dtype, const void *p, size_t stride, size_t cols) {
  return p && aligned_to(p, type_size(dtype)) && stride >= cols && stride <= ((size_t)1 << 40);
}

static int product4(int dtype, const void *x, size_t x_stride, const Matrix4 &m, int scale_dtype, const void *scales,
                    const void *book, const RowSource &src, void *y, size_t y_stride, hipStream_t s) {
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    return with_type(scale_dtype, [&](auto stag) {
      typedef typename decltype(stag)::type S;
      hipLaunchKernelGGL((product4_any_kernel<T, S>), dim3((unsigned)((m.out + 3) / 4), src.offsets ? src.experts + 1 : 1),
                         dim3(256), 0, s, static_cast<const T *>(x), (int64_t)x_stride, m,
                         static_cast<const S *>(scales), static_cast<const T *>(book), src, static_cast<T *>(y),
                         (int64_t)y_stride);
      return launched();
    });
  });
}

}  // namespace kmhip

using namespace kmhip;

KM_API int h2o4gpu_codebook4_quantize(int dtype, size_t out, size_t cols, int group, float top, const void *d_w,
                                      size_t w_stride, const void *d_codebook, void *d_codes, size_t codes_pitch,
                                      int scale_dtype, void *d_scales, void *stream) {
  if (!matrix_ok(dtype, out, cols, group, d_codes, codes_pitch, scale_dtype, d_scales, d_codebook) ||
      !strided_ok(dtype, d_w, w_stride, cols) || !(top > 0.f) || !isfinite(top))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    return with_type(scale_dtype, [&](auto stag) {
      typedef typename decltype(stag)::type S;
      hipLaunchKernelGGL((quantize4_kernel<T, S>), dim3((unsigned)((out + 3) / 4)), dim3(256), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T *>(d_w), (int64_t)w_stride,
                         (int64_t)out, (int)cols, group, top, static_cast<const T *>(d_codebook),
                         static_cast<uint8_t *>(d_codes), (int64_t)codes_pitch, static_cast<S *>(d_scales));
      return launched();
    });
  });
}

static Matrix4 matrix4(size_t out, size_t cols, int group, const void *codes, size_t pitch, size_t book_stride) {
  Matrix4 m;
  m.codes = static_cast<const uint8_t *>(codes);
  m.pitch = (int64_t)pitch;
  m.out = (int64_t)out;
  m.cols = (int)cols;
  m.group = group;
  m.groups = (int)((cols + group - 1) / group);
  m.book_stride = (int64_t)book_stride;
  return m;
}

KM_API int h2o4gpu_codebook4_product(int dtype, size_t rows, size_t out, size_t cols, int group, const void *d_x,
                                     size_t x_stride, const void *d_codes, size_t codes_pitch, int scale_dtype,
                                     const void *d_scales, const void *d_codebook, void *d_y, size_t y_stride,
                                     void *stream) {
  if (!matrix_ok(dtype, out, cols, group, d_codes, codes_pitch, scale_dtype, d_scales, d_codebook) ||
      rows > MOST_ROWS4)
    return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!strided_ok(dtype, d_x, x_stride, cols) || !strided_ok(dtype, d_y, y_stride, out)) return H2O4GPU_KMEANS_EARG;
  RowSource src;
  src.rows = (int64_t)rows;
  return product4(dtype, d_x, x_stride, matrix4(out, cols, group, d_codes, codes_pitch, 0), scale_dtype, d_scales,
                  d_codebook, src, d_y, y_stride, static_cast<hipStream_t>(stream));
}

KM_API int h2o4gpu_codebook4_experts_product(int dtype, size_t tokens, int top_k, int experts, size_t out,
                                             size_t cols, int group, const void *d_x, size_t x_stride,
                                             const void *d_codes, size_t codes_pitch, int scale_dtype,
                                             const void *d_scales, const void *d_codebook, size_t codebook_stride,
                                             const int *d_order, const int *d_offsets, void *d_y, size_t y_stride,
                                             void *stream) {
  if (!matrix_ok(dtype, out, cols, group, d_codes, codes_pitch, scale_dtype, d_scales, d_codebook) || experts < 1 ||
      experts > H2O4GPU_EXPERTS_MAX_EXPERTS || top_k < 1 || top_k > H2O4GPU_EXPERTS_MAX_TOP_K ||
      tokens > MOST_ROWS4 / (size_t)top_k || (codebook_stride != 0 && codebook_stride < 16) ||
      codebook_stride > ((size_t)1 << 32))
    return H2O4GPU_KMEANS_EARG;
  if (tokens == 0) return H2O4GPU_KMEANS_OK;
  if (!strided_ok(dtype, d_x, x_stride, cols) || !strided_ok(dtype, d_y, y_stride, out) || !d_order || !d_offsets ||
      !aligned_to(d_order, 4) || !aligned_to(d_offsets, 4))
    return H2O4GPU_KMEANS_EARG;
  RowSource src;
  src.order = d_order;
  src.offsets = d_offsets;
  src.top_k = top_k;
  src.experts = experts;
  src.rows = (int64_t)tokens * top_k;
  return product4(dtype, d_x, x_stride, matrix4(out, cols, group, d_codes, codes_pitch, codebook_stride), scale_dtype,
                  d_scales, d_codebook, src, d_y, y_stride, static_cast<hipStream_t>(stream));
}
