// Matrices of 4-bit codes: compressing one, and its product with tokens, alone or a matrix per expert.
#include "experts_common.h"
#include "mfma_traits.h"

#include <type_traits>

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

// The product on the matrix cores. x is the "A" operand (rows of the result tile: 16 tokens), the
// matrix the "B" operand (columns: 16 of y), so a lane holds one column of y and every scale it
// applies is its own column's:
//   A[i = lane % 16][k = VK * (lane / 16) + 0 .. VK-1], B[k likewise][j = lane % 16],
//   accumulator v: D[i = 4 * (lane / 16) + v][j = lane % 16].
// A wavefront takes 128 columns of the matrix at a time: lane (r, q) loads the 16 bytes of row r that
// hold group-of-32 number q, and a 4 x 4 transposition between the four lane groups and the four
// registers (four swaps) gives every lane 8 columns of each 32, so that no instruction mixes columns of
// two scales. Codes become values through a table of pairs in LDS, indexed by a whole byte: 256
// entries, each once per bank that a lane may read from, so the reads never collide (a table in
// registers takes 3.1 vector instructions a code, this one takes one and half a read). Products are
// exact in float, sums are float; the scale is applied to the sum over its group.
template <typename T>
struct Mfma4;

template <>
struct Mfma4<bfloat16_t> {
  typedef bfloat16_t vec __attribute__((ext_vector_type(8)));
  static constexpr int COPIES = 32;  // of the pair table: 4 bytes each
  static __device__ __forceinline__ floatx4 mma(const unsigned *a, const unsigned *b, floatx4 c) {
    vec va, vb;
    __builtin_memcpy(&va, a, 16);
    __builtin_memcpy(&vb, b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, vb, c, 0, 0, 0);
  }
};

template <>
struct Mfma4<float16_t> {
  typedef float16_t vec __attribute__((ext_vector_type(8)));
  static constexpr int COPIES = 32;
  static __device__ __forceinline__ floatx4 mma(const unsigned *a, const unsigned *b, floatx4 c) {
    vec va, vb;
    __builtin_memcpy(&va, a, 16);
    __builtin_memcpy(&vb, b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(va, vb, c, 0, 0, 0);
  }
};

template <>
struct Mfma4<float> {
  static constexpr int COPIES = 16;  // 8 bytes each
  static __device__ __forceinline__ floatx4 mma(const unsigned *a, const unsigned *b, floatx4 c) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
};

static const int TABLE_BYTES = 256 * 128;

// The same bytes at an address that is only aligned to its elements.
typedef unsigned uintx4_u __attribute__((ext_vector_type(4), aligned(2)));

// 8 values of x as 32-bit words; the last columns of a row with zeros behind them.
template <typename T>
__device__ __forceinline__ void load_x8(const T *at, unsigned (&w)[2 * sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; i++) {
    const uintx4_u v = reinterpret_cast<const uintx4_u *>(at)[i];
    w[4 * i] = v[0];
    w[4 * i + 1] = v[1];
    w[4 * i + 2] = v[2];
    w[4 * i + 3] = v[3];
  }
}
template <typename T>
__device__ __forceinline__ void load_x8_end(const T *at, int left, unsigned (&w)[2 * sizeof(T)]) {
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = i < left ? at[i] : (T)0.f;
  __builtin_memcpy(w, v, sizeof(v));
}

// 8 codes as 8 values: byte b of the word names a pair.
template <typename T>
__device__ __forceinline__ void decode8(const char *table, unsigned word, unsigned lane_at,
                                        unsigned (&w)[2 * sizeof(T)]) {
  const unsigned at0 = ((word << 7) & 0x7f80u) | lane_at, at1 = ((word >> 1) & 0x7f80u) | lane_at;
  const unsigned at2 = ((word >> 9) & 0x7f80u) | lane_at, at3 = ((word >> 17) & 0x7f80u) | lane_at;
  typedef typename std::conditional<sizeof(T) == 4, uint2, unsigned>::type Pair;
  const Pair p[4] = {*reinterpret_cast<const Pair *>(table + at0), *reinterpret_cast<const Pair *>(table + at1),
                     *reinterpret_cast<const Pair *>(table + at2), *reinterpret_cast<const Pair *>(table + at3)};
  __builtin_memcpy(w, p, sizeof(p));
}

// A scale of 32 or of 16 bits, the latter of either type.
__device__ __forceinline__ float scale_value(float v, bool) { return v; }
__device__ __forceinline__ float scale_value(uint16_t v, bool brain) {
  float16_t h;
  __builtin_memcpy(&h, &v, 2);
  return brain ? __uint_as_float((unsigned)v << 16) : (float)h;
}

struct Product4Args {
  Matrix4 m;
  bool brain;                // 16-bit scales are bfloat16
  RowSource src;
  int64_t xs, ys;
  unsigned per_scale;        // how many 32s (FINE) or 128s of columns share a scale
  unsigned per_scale_magic;  // ceil(2^32 / per_scale); 0 where that is 1
};

// What a wavefront has in flight: U times 128 columns of the matrix.
template <typename T, typename S, int MT, int NT, int U, bool FINE>
struct Stage {
  uint4 words[U][NT];
  S scale[U][NT][FINE ? 4 : 1];  // as they lie in memory: nothing waits for them before they are used
  unsigned x[U][MT][4][2 * sizeof(T)];
};

// acc += scale * (x times 128 columns of the matrix's transpose).
template <typename T, typename S, int MT, int NT, int U, bool FINE>
__device__ __forceinline__ void multiply(const Stage<T, S, MT, NT, U, FINE> &st, int u, const char *table,
                                         unsigned lane_at, bool brain, floatx4 (&acc)[MT][NT]) {
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const uint4 w = st.words[u][t];
    const auto s02 = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false);
    const auto s13 = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
    const auto d01 = __builtin_amdgcn_permlane16_swap(s02[0], s13[0], false, false);
    const auto d23 = __builtin_amdgcn_permlane16_swap(s02[1], s13[1], false, false);
    const unsigned d[4] = {d01[0], d01[1], d23[0], d23[1]};
    floatx4 part[MT] = {};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      unsigned b[2 * sizeof(T)];
      decode8<T>(table, d[i], lane_at, b);
#pragma unroll
      for (int m = 0; m < MT; m++) {
        part[m] = Mfma4<T>::mma(st.x[u][m][i], b, part[m]);
        if (FINE || i == 3) {
#pragma unroll
          for (int v = 0; v < 4; v++)
            acc[m][t][v] = fmaf(scale_value(st.scale[u][t][FINE ? i : 0], brain), part[m][v], acc[m][t][v]);
          part[m] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
      }
    }
  }
}

// A workgroup has 16 * NT columns of y and 16 * MT rows of it at a time; its wavefronts share the
// columns of the matrix, 128 * U to each in turn, the next ones on their way while the last are
// multiplied, and add their sums up in LDS. Rows of x behind the last one and rows of the matrix behind
// y's last column are read from the nearest that is there: their results are not written. FINE: scales
// change every 32 columns, not only every 128.
template <typename T, typename S, int MT, int NT, int U, bool FINE>
__global__ __launch_bounds__(512) void product4_kernel(const T *x, const S *scales, const T *books, T *y,
                                                       Product4Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  typedef Stage<T, S, MT, NT, U, FINE> Stg;
  constexpr int P = 2 * sizeof(T);  // bytes of a pair
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  float *red = reinterpret_cast<float *>(lds + TABLE_BYTES);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NT);

  int e = 0;
  int64_t lo = 0, hi = a.src.rows;
  if (a.src.offsets) {
    const int E = a.src.experts;
    if (blockIdx.y == gridDim.y - 1) {  // zeros for the rows that have no expert
      lo = a.src.offsets[E];
      for (int64_t p = lo + blockIdx.z * waves + wave; p < hi; p += gridDim.z * waves)
        for (int c = lane; c < 16 * NT; c += 64)
          if (n0 + c < a.m.out) y[p * a.ys + n0 + c] = (T)0.f;
      return;
    }
    if ((int)gridDim.y - 1 == E) {
      e = blockIdx.y;
      lo = a.src.offsets[e];
      hi = a.src.offsets[e + 1];
    } else {  // fewer rows than experts: the workgroups of an expert's first row have all of its rows
      int *found = reinterpret_cast<int *>(red);
      if (threadIdx.x == 0) found[0] = -1;
      __syncthreads();
      const int p = blockIdx.y;
      for (int i = threadIdx.x; i < E; i += blockDim.x) {
        const int from = a.src.offsets[i], to = a.src.offsets[i + 1];
        if (from == p && to > p) {
          found[0] = i;
          found[1] = to;
        }
      }
      __syncthreads();
      e = __builtin_amdgcn_readfirstlane(found[0]);
      lo = p;
      hi = e >= 0 ? found[1] : lo;
      __syncthreads();
    }
  }
  lo += (int64_t)blockIdx.z * (16 * MT);
  if (lo >= hi) return;

  const unsigned lane_at = (lane & (Mfma4<T>::COPIES - 1)) * P;
  const int cols = a.m.cols, full = cols >> 7;
  const uint8_t *code[NT];
  const S *scale[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int64_t n = n0 + 16 * t + r < a.m.out ? n0 + 16 * t + r : a.m.out - 1;
    code[t] = a.m.codes + (e * a.m.out + n) * a.m.pitch;
    scale[t] = scales + (e * a.m.out + n) * a.m.groups;
  }
  const T *row[MT];
  const auto rows_from = [&](int64_t first) {
#pragma unroll
    for (int t = 0; t < MT; t++) {
      const int64_t p = first + 16 * t + r < hi ? first + 16 * t + r : hi - 1;
      row[t] = x + (a.src.order ? a.src.order[p] / a.src.top_k : p) * a.xs;
    }
  };
  const auto load_scales = [&](Stg &st, int u, int sub) {
#pragma unroll
    for (int i = 0; i < (FINE ? 4 : 1); i++) {
      const unsigned unit = FINE ? sub * 4 + i : sub;
      unsigned g = a.per_scale_magic ? __umulhi(unit, a.per_scale_magic) : unit;
      g = g < (unsigned)a.m.groups ? g : a.m.groups - 1;
#pragma unroll
      for (int t = 0; t < NT; t++) st.scale[u][t][i] = scale[t][g];
    }
  };
  const auto fetch = [&](Stg &st, int s0) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int sub = s0 + u < full ? s0 + u : full - 1;
#pragma unroll
      for (int t = 0; t < NT; t++)
        st.words[u][t] = *reinterpret_cast<const uint4 *>(code[t] + ((int64_t)sub * 64 + q * 16));
      load_scales(st, u, sub);
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) load_x8<T>(row[t] + (sub * 128 + 32 * i + 8 * q), st.x[u][t][i]);
    }
  };
  const auto table = [&]() {  // thread t writes copies of entry t / 2
    const T *book = books + e * a.m.book_stride;
    for (int i = threadIdx.x; i < 512; i += blockDim.x) {
      const int byte = i >> 1;
      T pair[16 / sizeof(T)];
#pragma unroll
      for (int c = 0; c < (int)(16 / sizeof(T)); c += 2) {
        pair[c] = book[byte & 15];
        pair[c + 1] = book[byte >> 4];
      }
      uint4 four;
      __builtin_memcpy(&four, pair, 16);
#pragma unroll
      for (int c = 0; c < 4; c++) *reinterpret_cast<uint4 *>(lds + i * 64 + c * 16) = four;
    }
    __syncthreads();
  };

  bool have_table = false;
  for (; lo < hi; lo += (int64_t)gridDim.z * (16 * MT)) {
    rows_from(lo);
    floatx4 acc[MT][NT] = {};
    const int step = waves * U;
    Stg st[2];
    int s = wave * U;
    if (s < full) fetch(st[0], s);
    if (!have_table) table();
    have_table = true;
    while (s < full) {
      if (s + step < full) fetch(st[1], s + step);
#pragma unroll
      for (int u = 0; u < U; u++)
        if (s + u < full) multiply(st[0], u, lds, lane_at, a.brain, acc);
      s += step;
      if (s >= full) break;
      if (s + step < full) fetch(st[0], s + step);
#pragma unroll
      for (int u = 0; u < U; u++)
        if (s + u < full) multiply(st[1], u, lds, lane_at, a.brain, acc);
      s += step;
    }
    if ((cols & 127) && wave == full % waves) {  // the columns behind the last whole 128
      Stage<T, S, MT, NT, 1, FINE> end;
      const int64_t last = a.m.pitch - 16, at = (int64_t)full * 64 + q * 16;
#pragma unroll
      for (int t = 0; t < NT; t++) end.words[0][t] = *reinterpret_cast<const uint4 *>(code[t] + (at < last ? at : last));
#pragma unroll
      for (int i = 0; i < (FINE ? 4 : 1); i++) {
        const unsigned unit = FINE ? full * 4 + i : full;
        unsigned g = a.per_scale_magic ? __umulhi(unit, a.per_scale_magic) : unit;
        g = g < (unsigned)a.m.groups ? g : a.m.groups - 1;
#pragma unroll
        for (int t = 0; t < NT; t++) end.scale[0][t][i] = scale[t][g];
      }
#pragma unroll
      for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int k = full * 128 + 32 * i + 8 * q;
          load_x8_end<T>(row[t] + k, cols - k, end.x[0][t][i]);
        }
      multiply(end, 0, lds, lane_at, a.brain, acc);
    }
    // the wavefronts' sums, in their order
#pragma unroll
    for (int m = 0; m < MT; m++) {
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int v = 0; v < 4; v++) red[(wave * (4 * NT) + 4 * t + v) * 64 + lane] = acc[m][t][v];
      __syncthreads();
      for (int i = threadIdx.x; i < 4 * NT * 64; i += blockDim.x) {
        // i = (token, column): 16 neighbours write 16 columns of one row
        const int token = i / (16 * NT), c = i % (16 * NT);
        const int64_t p = lo + 16 * m + token, n = n0 + c;
        if (p < hi && n < a.m.out) {
          const int at = (4 * (c >> 4) + (token & 3)) * 64 + (token >> 2) * 16 + (c & 15);
          float sum = 0.f;
          for (int w = 0; w < waves; w++) sum += red[w * (4 * NT * 64) + at];
          y[p * a.ys + n] = (T)sum;
        }
      }
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

template <typename T, typename S, int MT, int NT, int U, bool FINE>
static int launch_product4(const T *x, const S *scales, const T *book, T *y, const Product4Args &a, int waves,
                           hipStream_t s) {
  const size_t lds = TABLE_BYTES + (size_t)waves * 4 * NT * 64 * sizeof(float);
  const void *kernel = reinterpret_cast<const void *>(product4_kernel<T, S, MT, NT, U, FINE>);
  KM_TRY(ensure_dynamic_lds(kernel, lds));
  const unsigned gx = (unsigned)((a.m.out + 16 * NT - 1) / (16 * NT));
  unsigned gy = 1, gz = 1;
  const int64_t tiles = (a.src.rows + 16 * MT - 1) / (16 * MT);
  if (a.src.offsets)
    gy = (unsigned)(a.src.rows < a.src.experts ? a.src.rows : a.src.experts) + 1;
  else  // a workgroup that has several tiles of tokens makes its table once
    gz = (unsigned)(tiles < 256 ? tiles : 256);
  hipLaunchKernelGGL((product4_kernel<T, S, MT, NT, U, FINE>), dim3(gx, gy, gz), dim3(64 * waves), lds, s, x, scales,
                     book, y, a);
  return launched();
}

static int product4(int dtype, const void *x, size_t x_stride, const Matrix4 &m, int scale_dtype, const void *scales,
                    const void *book, const RowSource &src, void *y, size_t y_stride, hipStream_t s) {
  Product4Args a;
  a.m = m;
  a.brain = scale_dtype == H2O4GPU_EXPERTS_BFLOAT16;
  a.src = src;
  a.xs = (int64_t)x_stride;
  a.ys = (int64_t)y_stride;
  const bool fine = m.group % 128 != 0;
  const unsigned unit = fine ? 32 : 128;
  a.per_scale = (unsigned)m.group / unit;
  const unsigned most = (unsigned)m.cols / unit + 1;
  if (a.per_scale > most) a.per_scale = most;
  a.per_scale_magic = a.per_scale == 1 ? 0u : (unsigned)((0x100000000ull + a.per_scale - 1) / a.per_scale);
  const int subs = (m.cols + 127) / 128;
  int waves = 8;
  while (waves > 1 && waves / 2 >= subs) waves /= 2;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    const auto with_scales = [&](auto *ts) {
      typedef typename std::remove_const<typename std::remove_pointer<decltype(ts)>::type>::type S;
      const T *tx = static_cast<const T *>(x), *tb = static_cast<const T *>(book);
      T *ty = static_cast<T *>(y);
      return fine ? launch_product4<T, S, 1, 1, 2, true>(tx, ts, tb, ty, a, waves, s)
                  : launch_product4<T, S, 1, 1, 2, false>(tx, ts, tb, ty, a, waves, s);
    };
    return scale_dtype == H2O4GPU_EXPERTS_FLOAT32 ? with_scales(static_cast<const float *>(scales))
                                                  : with_scales(static_cast<const uint16_t *>(scales));
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
