// Microscaled 4-bit numbers: blocks of 32 elements with one sign, two exponent and one mantissa bit (0, 0.5, 1,
// 1.5, 2, 3, 4, 6) share a power of two, 2^(byte - 127). Numbers into them and back, and products of two such
// matrices on the scaled matrix instructions, which multiply 128 columns of both in the time of 32 in 16 bits.
//
// A matrix lies in memory in rows: codes two to a byte, the even column in the low half, 128 bytes (256 columns)
// or a multiple to a row; scales 16 bytes for 512 columns, the byte of the block b of these 16 at 4 * (b % 4) + b / 4:
// lane group g of a matrix instruction multiplies block g of its 128 columns, and has the scales of four
// instructions in one word. Behind a row's last column lie zeros (codes and scales).
#include "product_thin.h"

namespace kmhip {
namespace {

constexpr size_t MAX_SIDE = (size_t)1 << 30;

__host__ __device__ inline size_t codes_pitch(size_t cols) { return (cols + 255) / 256 * 128; }
__host__ __device__ inline size_t scales_pitch(size_t cols) { return (cols + 511) / 512 * 16; }
__host__ __device__ inline unsigned scale_place(unsigned block) {
  return block / 16 * 16 + block % 4 * 4 + block % 16 / 4;
}
// The element a code's low four bits stand for: sign, two bits of exponent, one of mantissa. The bits of 2 m, 2 m + 1
// halves put where a float has its own make 2^-126 times as much (and 0.5 a denormal number that the product mends).
__device__ __forceinline__ float element(unsigned code) {
  const float m = __uint_as_float((code & 7) << 22) * 0x1p126f;
  return __uint_as_float(__float_as_uint(m) | (code & 8) << 28);
}
__device__ __forceinline__ float power_of(unsigned byte) {
  return byte == 255 ? __builtin_nanf("") : __uint_as_float(byte ? byte << 23 : 0x400000u);
}

// One thread: eight columns, a word of codes; four threads a block, which share its largest magnitude. A block's power of
// two is that of the largest magnitude over 4, so that it lands in [4, 8), where 6 is the largest element and what is
// beyond stays 6. Magnitudes are compared as their bits, in which NaN and infinities are the largest: their block's scale
// is 255, not a number. Bound by memory, 1024 bytes of 16-bit elements in and 272 out a wavefront: two words a thread,
// both loads on their way at once, and no other pass. 11003 x 8190 float16 (228 MB in all) take 42 us, 5.5 TB/s out of a
// warm cache; with one word a thread 47, with four 43 (8192 x 8192 28, 30 and 32). 64 x 4096 take a launch, 4 us.
template <typename T, int UNROLL>
__global__ __launch_bounds__(256) void quantize_kernel(const T *x, size_t x_stride, unsigned cols, size_t words,
                                                       unsigned row_words, unsigned *codes, unsigned char *scales,
                                                       unsigned scales_row, unsigned first_block) {
  const size_t base = (size_t)(first_block + blockIdx.x) * (256 * UNROLL) + threadIdx.x;
  u32x4 in[UNROLL][sizeof(T) / 2];
  size_t row[UNROLL];
  unsigned word[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const size_t at = base + u * 256;
    row[u] = at / row_words;
    word[u] = (unsigned)(at - row[u] * row_words);
    const int left = at < words ? (int)cols - (int)word[u] * 8 : 0;
    const T *p = x + row[u] * x_stride + word[u] * 8;
#pragma unroll
    for (int h = 0; h < (int)sizeof(T) / 2; ++h)
      in[u][h] = load_piece(p + h * (16 / sizeof(T)), left - h * (int)(16 / sizeof(T)));
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(in[u][i / 4][i % 4]);
      } else {
        const unsigned short bits = (unsigned short)(in[u][0][i / 2] >> (16 * (i & 1)));
        v[i] = (float)__builtin_bit_cast(T, bits);
      }
    }
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned m = __float_as_uint(v[i]) & 0x7fffffffu;
      most = m > most ? m : most;
    }
#pragma unroll
    for (int d = 1; d < 4; d *= 2) {
      const unsigned other = __shfl_xor(most, d);
      most = other > most ? other : most;
    }
    const unsigned e = most >> 23, byte = e == 255 ? 255 : e > 2 ? e - 2 : 0;
    unsigned out = 0;
#if defined(__HIP_DEVICE_COMPILE__)
    // rounds to the nearest, a tie to the even mantissa, and saturates
    const float power = __uint_as_float(byte ? byte << 23 : 0x400000u);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[0], v[1], power, 0);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[2], v[3], power, 1);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[4], v[5], power, 2);
    out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(out, v[6], v[7], power, 3);
#endif
    if (byte == 255) out = 0;
    if (base + u * 256 < words) {
      codes[base + u * 256] = out;
      if ((word[u] & 3) == 0) {
        unsigned char *s = scales + row[u] * scales_row + scale_place(word[u] / 4);
        s[0] = (unsigned char)byte;
        // the last 256 columns of a row that is no multiple of 512: the other half's bytes
        if ((word[u] & 63) < 32 && (word[u] | 31) == row_words - 1) s[2] = 0;
      }
    }
  }
}

// One thread: a word of codes, eight numbers of a row side by side. Bound by what it writes: 11003 x 8190 float16 40 us, 5.6
// TB/s.
template <typename T>
__global__ __launch_bounds__(256) void dequantize_kernel(const unsigned *codes, const unsigned char *scales, unsigned cols,
                                                         size_t words, unsigned row_words, unsigned scales_row, T *out,
                                                         size_t out_stride, unsigned first_block) {
  const size_t at = (size_t)(first_block + blockIdx.x) * 256 + threadIdx.x;
  if (at >= words) return;
  const size_t row = at / row_words;
  const unsigned word = (unsigned)(at - row * row_words);
  if (word * 8 >= cols) return;
  const unsigned code = codes[row * (codes_pitch(cols) / 4) + word];
  const float power = power_of(scales[row * scales_row + scale_place(word / 4)]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = element(code >> (4 * i)) * power;
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(v[i]));  // (as one instruction with a conversion to float16, -0 would become 0)
#endif
  }
  T *o = out + row * out_stride + word * 8;
  const int left = (int)cols - (int)word * 8;
  if (left >= 8) {
    typedef typename Beside<T, 8>::vector eight;
    const eight all = {(T)v[0], (T)v[1], (T)v[2], (T)v[3], (T)v[4], (T)v[5], (T)v[6], (T)v[7]};
    store_beside<T, 8>(o, all);
  } else {
    store_four(o, f32x4{v[0], v[1], v[2], v[3]}, left);
    store_four(o + 4, f32x4{v[4], v[5], v[6], v[7]}, left - 4);
  }
}

// Codes and scales that come in plain rows, into the layout above: a word of codes a thread, once for a matrix
// (8192 x 8192 33 us).
__global__ __launch_bounds__(256) void layout_kernel(const unsigned char *in, size_t in_pitch, const unsigned char *in_scales,
                                                     unsigned cols, size_t words, unsigned row_words, unsigned *codes,
                                                     unsigned char *scales, unsigned scales_row, unsigned first_block) {
  const size_t at = (size_t)(first_block + blockIdx.x) * 256 + threadIdx.x;
  if (at >= words) return;
  const size_t row = at / row_words;
  const unsigned word = (unsigned)(at - row * row_words);
  unsigned out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned col = word * 8 + 2 * i;
    if (col < cols) {
      unsigned two = in[row * in_pitch + col / 2];
      if (col + 1 == cols) two &= 15;
      out |= two << (8 * i);
    }
  }
  codes[at] = out;
  if ((word & 3) == 0) {
    const unsigned block = word / 4, blocks = (cols + 31) / 32;
    unsigned char *s = scales + row * scales_row + scale_place(block);
    s[0] = block < blocks ? in_scales[row * blocks + block] : 0;
    if ((word & 63) < 32 && (word | 31) == row_words - 1) s[2] = 0;
  }
}

struct FourArgs {
  const unsigned char *x, *x_scales, *w, *w_scales;
  void *y;
  size_t y_stride;
  const int *order, *offsets;  // with experts only; order: x's row of y's row p is order[p] / top_k (none: p)
  int top_k, experts;          // experts 0: one matrix
  int rows, out, cols;
};

template <typename T>
int launch_four(const FourArgs &a, size_t x_rows, hipStream_t stream) {
  const size_t pitch = codes_pitch(a.cols);
  const Way way = way_of_four(a.rows, a.experts, a.out, a.cols, pitch, a.order != nullptr, x_rows);
  if (way == FEW_ROWS || way == KEPT) {
    ThinArgs t = {};
    t.x = (const char *)a.x, t.w = (const char *)a.w, t.x_scales = a.x_scales, t.w_scales = a.w_scales, t.c = a.y;
    t.x_stride = t.w_stride = pitch, t.w_expert = pitch * a.out, t.scales_stride = scales_pitch(a.cols);
    t.c_stride = a.y_stride, t.order = a.order, t.offsets = a.offsets, t.top_k = a.top_k;
    t.experts = a.experts, t.rows = a.rows, t.n = a.out, t.k = (int)((a.cols + 127) / 128 * 32);
    if (way == KEPT) return launch_kept<T>(t, stream);
    return launch_thin<Four, T, true>(t, stream);
  }
  PipeArgs p = {};
  p.x = (const char *)a.x, p.w = (const char *)a.w, p.x_scales = a.x_scales, p.w_scales = a.w_scales, p.c = a.y;
  p.x_stride = p.w_stride = pitch, p.w_expert = pitch * a.out, p.scales_stride = scales_pitch(a.cols);
  p.c_stride = a.y_stride, p.x_bytes = x_rows * pitch;
  p.order = a.order, p.offsets = a.offsets, p.top_k = a.top_k, p.experts = a.experts;
  p.rows = a.rows, p.n = a.out, p.k = (int)(pitch / 2);
  return a.order ? launch_large<Four, T, FORWARD, true>(p, way, stream)
                 : launch_large<Four, T, FORWARD, false>(p, way, stream);
}

bool sized(size_t rows, size_t cols) { return cols >= 1 && cols <= MAX_SIDE && rows <= ((size_t)1 << 40) / codes_pitch(cols); }

}  // namespace
}  // namespace kmhip

using namespace kmhip;

KM_API size_t h2o4gpu_microscale4_codes_pitch(size_t cols) { return cols < 1 || cols > MAX_SIDE ? 0 : codes_pitch(cols); }
KM_API size_t h2o4gpu_microscale4_scales_pitch(size_t cols) {
  return cols < 1 || cols > MAX_SIDE ? 0 : scales_pitch(cols);
}

KM_API int h2o4gpu_microscale4_quantize(int dtype, size_t rows, size_t cols, const void *d_x, size_t x_stride,
                                        void *d_codes, void *d_scales, void *stream) {
  if (!known_type(dtype) || !sized(rows, cols)) return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!d_x || !d_codes || !d_scales || (rows > 1 && x_stride < cols) ||
      !aligned_to(d_x, type_size(dtype)) || !aligned_to(d_codes, 16) ||
      !aligned_to(d_scales, 16))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    constexpr int UNROLL = 2;
    const unsigned row_words = (unsigned)(codes_pitch(cols) / 4);
    const size_t words = rows * row_words, blocks = (words + 256 * UNROLL - 1) / (256 * UNROLL);
    return in_launches(blocks, [&](unsigned first, unsigned here) {
      hipLaunchKernelGGL((quantize_kernel<T, UNROLL>), dim3(here), dim3(256), 0, static_cast<hipStream_t>(stream),
                         static_cast<const T *>(d_x), x_stride, (unsigned)cols, words, row_words,
                         static_cast<unsigned *>(d_codes), static_cast<unsigned char *>(d_scales),
                         (unsigned)scales_pitch(cols), first);
      return launched();
    });
  });
}

KM_API int h2o4gpu_microscale4_dequantize(int dtype, size_t rows, size_t cols, const void *d_codes, const void *d_scales,
                                          void *d_out, size_t out_stride, void *stream) {
  if (!known_type(dtype) || !sized(rows, cols)) return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!d_out || !d_codes || !d_scales || (rows > 1 && out_stride < cols) ||
      !aligned_to(d_out, type_size(dtype)) || !aligned_to(d_codes, 16) ||
      !aligned_to(d_scales, 16))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    const unsigned row_words = (unsigned)((cols + 7) / 8);
    const size_t words = rows * row_words;
    return in_launches((words + 255) / 256, [&](unsigned first, unsigned here) {
      hipLaunchKernelGGL((dequantize_kernel<T>), dim3(here), dim3(256), 0, static_cast<hipStream_t>(stream),
                         static_cast<const unsigned *>(d_codes), static_cast<const unsigned char *>(d_scales),
                         (unsigned)cols, words, row_words, (unsigned)scales_pitch(cols), static_cast<T *>(d_out),
                         out_stride, first);
      return launched();
    });
  });
}

KM_API int h2o4gpu_microscale4_layout(size_t rows, size_t cols, const void *d_codes, size_t codes_stride,
                                      const void *d_scales, void *d_laid_codes, void *d_laid_scales, void *stream) {
  if (!sized(rows, cols)) return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!d_codes || !d_scales || !d_laid_codes || !d_laid_scales || codes_stride < (cols + 1) / 2 ||
      !aligned_to(d_laid_codes, 16) || !aligned_to(d_laid_scales, 16))
    return H2O4GPU_KMEANS_EARG;
  const unsigned row_words = (unsigned)(codes_pitch(cols) / 4);
  const size_t words = rows * row_words;
  return in_launches((words + 255) / 256, [&](unsigned first, unsigned here) {
    hipLaunchKernelGGL(layout_kernel, dim3(here), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const unsigned char *>(d_codes), codes_stride,
                       static_cast<const unsigned char *>(d_scales), (unsigned)cols, words, row_words,
                       static_cast<unsigned *>(d_laid_codes), static_cast<unsigned char *>(d_laid_scales),
                       (unsigned)scales_pitch(cols), first);
    return launched();
  });
}

namespace {
int four_product(int dtype, FourArgs a, size_t x_rows, size_t rows, size_t out, size_t cols, void *stream) {
  if (!known_type(dtype) || !sized(rows, cols) || out < 1 || out > MAX_SIDE || rows > (size_t)INT_MAX - 65536)
    return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!a.x || !a.x_scales || !a.w || !a.w_scales || !a.y || (rows > 1 && a.y_stride < out)) return H2O4GPU_KMEANS_EARG;
  for (const void *p : {a.x, a.x_scales, a.w, a.w_scales})
    if (!aligned_to(p, 16)) return H2O4GPU_KMEANS_EARG;
  if (!aligned_to(a.y, type_size(dtype))) return H2O4GPU_KMEANS_EARG;
  a.rows = (int)rows, a.out = (int)out, a.cols = (int)cols;
  return with_type(dtype, [&](auto tag) {
    return launch_four<typename decltype(tag)::type>(a, x_rows, static_cast<hipStream_t>(stream));
  });
}
}  // namespace

KM_API int h2o4gpu_microscale4_product(int dtype, size_t rows, size_t out, size_t cols, const void *d_x,
                                       const void *d_x_scales, const void *d_w, const void *d_w_scales, void *d_y,
                                       size_t y_stride, void *stream) {
  FourArgs a = {};
  a.x = static_cast<const unsigned char *>(d_x), a.x_scales = static_cast<const unsigned char *>(d_x_scales);
  a.w = static_cast<const unsigned char *>(d_w), a.w_scales = static_cast<const unsigned char *>(d_w_scales);
  a.y = d_y, a.y_stride = y_stride;
  return four_product(dtype, a, rows, rows, out, cols, stream);
}

KM_API int h2o4gpu_microscale4_experts_product(int dtype, size_t tokens, int top_k, int experts, size_t out, size_t cols,
                                               const void *d_x, const void *d_x_scales, const void *d_w,
                                               const void *d_w_scales, const int *d_order, const int *d_offsets, void *d_y,
                                               size_t y_stride, void *stream) {
  if (experts < 1 || experts > H2O4GPU_EXPERTS_MAX_EXPERTS || top_k < 1 || top_k > H2O4GPU_EXPERTS_MAX_TOP_K ||
      tokens > (size_t)INT_MAX)
    return H2O4GPU_KMEANS_EARG;
  if (tokens && !d_offsets) return H2O4GPU_KMEANS_EARG;
  FourArgs a = {};
  a.x = static_cast<const unsigned char *>(d_x), a.x_scales = static_cast<const unsigned char *>(d_x_scales);
  a.w = static_cast<const unsigned char *>(d_w), a.w_scales = static_cast<const unsigned char *>(d_w_scales);
  a.y = d_y, a.y_stride = y_stride;
  a.order = d_order, a.offsets = d_offsets, a.top_k = top_k, a.experts = experts;
  return four_product(dtype, a, d_order ? tokens : tokens * top_k, tokens * top_k, out, cols, stream);
}
