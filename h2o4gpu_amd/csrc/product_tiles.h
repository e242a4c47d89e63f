// Tiles of matrix products on gfx950: how an operand's stage lies in LDS, how a wavefront reads its part of it
// for the matrix instructions, and which rows a tile of a ragged product holds.
//
// A product here is C[m][n] = sum over k of X[m][k] * W[n][k]. An operand comes with k contiguous ("rows") or with
// m or n contiguous ("columns": k is the row of the matrix in memory). Everything moves in pieces of 16 bytes,
// and a stage of an operand tile is 128 bytes of k for each of its rows, in either order.
#pragma once

#include <limits.h>

#include "experts_common.h"
#include "product_rules.h"

namespace kmhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// acc[4 g + j of 16 n][lane % 16 of 16 m] += w's fragment times x's. A fragment is a piece of each lane's row
// (lane % 16): the elements k = EPP * (lane / 16) + i of a step of 4 * EPP. float32 has no instruction of that
// shape; four with one element a lane add up the same k.
__device__ __forceinline__ void mfma_piece(f32x4 &acc, u32x4 w, u32x4 x, Tag<bfloat16_t>) {
#if defined(__HIP_DEVICE_COMPILE__)
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), acc, 0, 0, 0);
#endif
}
__device__ __forceinline__ void mfma_piece(f32x4 &acc, u32x4 w, u32x4 x, Tag<float16_t>) {
#if defined(__HIP_DEVICE_COMPILE__)
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, x), acc, 0, 0, 0);
#endif
}
__device__ __forceinline__ void mfma_piece(f32x4 &acc, u32x4 w, u32x4 x, Tag<float>) {
#if defined(__HIP_DEVICE_COMPILE__)
  const f32x4 a = __builtin_bit_cast(f32x4, w), b = __builtin_bit_cast(f32x4, x);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
#endif
}

// Where the pieces of a stage of R rows lie. Slots are filled in order by consecutive lanes; which piece a slot
// holds is turned by its row (rows) or by its k (columns), so that the lanes of one read fall into different banks.
template <typename T, int R, bool COLUMNS>
struct OperandTile {
  static constexpr int EPP = 16 / (int)sizeof(T);  // elements of a piece
  static constexpr int KS = 8 * EPP;               // k of a stage
  static constexpr int SLOTS = R * 8;
  static constexpr int PER_K = R / EPP;            // pieces of one k (columns)

  static __device__ __forceinline__ int turn(int k) {
    // two bytes: a read takes pieces 2 b and 2 b + 1 of the k's 8 g + 4 h + 0..3 for g = 0..3
    return (sizeof(T) == 2 ? 2 * ((k & 3) + 4 * ((k >> 3) & 1)) : 4 * ((k >> 2) & 3)) & (PER_K - 1);
  }
  // slot -> first row and first k of its piece within the stage
  static __device__ __forceinline__ void place(int slot, int &row, int &k) {
    if (COLUMNS) {
      k = slot / PER_K;
      row = ((slot % PER_K) ^ turn(k)) * EPP;
    } else {
      row = slot / 8;
      k = ((slot % 8) ^ (row & 7)) * EPP;
    }
  }
  // the lane's fragment of rows 16 block .. + 15 for step 0 or 1 of the stage
  static __device__ __forceinline__ u32x4 fragment(const char *lds, int lane, int block, int step) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!COLUMNS) {
      const int row = block * 16 + i;
      return *reinterpret_cast<const u32x4 *>(lds + (row * 8 + ((step * 4 + g) ^ (row & 7))) * 16);
    } else if constexpr (sizeof(T) == 2) {
      u32x4 out;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = step * 32 + 8 * g + 4 * h + (i >> 2), c = 2 * block + ((i & 3) >> 1);
        const char *at = lds + (k * PER_K + (c ^ turn(k))) * 16 + (i & 1) * 8;
#if defined(__HIP_DEVICE_COMPILE__)
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        const s16x4 four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4 *)(const_cast<char *>(at)));
        const u32x2 two = __builtin_bit_cast(u32x2, four);
        out[2 * h] = two[0];
        out[2 * h + 1] = two[1];
#else
        out[2 * h] = out[2 * h + 1] = (unsigned)(size_t)at;
#endif
      }
      return out;
    } else {
      u32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = step * 16 + 4 * g + j, c = 4 * block + (i >> 2);
        out[j] = *reinterpret_cast<const unsigned *>(lds + (k * PER_K + (c ^ turn(k))) * 16 + (i & 3) * 4);
      }
      return out;
    }
  }
};

// Words from a buffer, zeros behind its end; all addresses are multiples of 4.
__device__ __forceinline__ u32x4 buffer_words(const char *from, unsigned size, unsigned at) {
  u32x4 v = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
  v = __builtin_amdgcn_raw_buffer_load_b128(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from), 0, (int)size, 0x00020000), (int)at, 0, 0);
#endif
  return v;
}
__device__ __forceinline__ unsigned buffer_word(const char *from, unsigned size, unsigned at) {
  unsigned v = 0;
#if defined(__HIP_DEVICE_COMPILE__)
  v = __builtin_amdgcn_raw_buffer_load_b32(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from), 0, (int)size, 0x00020000), (int)at, 0, 0);
#endif
  return v;
}
// A piece out of five words, the last beside: it begins `by` bytes, 0 or 2, behind the first.
__device__ __forceinline__ u32x4 shifted(u32x4 v, unsigned last, unsigned by) {
  by *= 8;
  return u32x4{__builtin_amdgcn_alignbit(v[1], v[0], by), __builtin_amdgcn_alignbit(v[2], v[1], by),
               __builtin_amdgcn_alignbit(v[3], v[2], by), __builtin_amdgcn_alignbit(last, v[3], by)};
}
// All bits of a piece's first `elements`.
template <typename T>
__device__ __forceinline__ u32x4 first_of(int elements) {
  u32x4 keep;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int bytes = elements * (int)sizeof(T) - 4 * i;
    keep[i] = bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : 0xffffu;
  }
  return keep;
}

// A whole piece, from any address that a T may have. The memory unit takes words at multiples of 4 as fast as at multiples
// of 16, and others three times slower: of 2-byte elements that lie between words (`halves`: some of the caller's do), the
// words that hold them are loaded and shifted. No word is touched that holds none of the piece.
template <typename T>
__device__ __forceinline__ u32x4 load_whole(const T *p, bool halves) {
  struct __attribute__((packed, aligned(4))) Words {
    u32x4 v;
  };
  if constexpr (sizeof(T) == 4) {
    return reinterpret_cast<const Words *>(p)->v;
  } else {
    if (!halves) return reinterpret_cast<const Words *>(p)->v;
    const size_t at = (size_t)p;
    return shifted(reinterpret_cast<const Words *>(at & ~(size_t)3)->v,
                   *reinterpret_cast<const unsigned *>((at + 14) & ~(size_t)3), (unsigned)(at & 2));
  }
}
// A piece of which the first `valid` elements exist, zeros behind (and all zeros for valid <= 0), from any address
// that a T may have.
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T *p, int valid) {
  constexpr int EPP = 16 / (int)sizeof(T);
  if (valid >= EPP) return load_whole(p, true);
  u32x4 out = {0, 0, 0, 0};
  if (valid > 0) {
#pragma unroll
    for (int i = 0; i < EPP; ++i) {
      if (i < valid) {
        if constexpr (sizeof(T) == 4)
          out[i] = *reinterpret_cast<const unsigned *>(p + i);
        else
          out[i / 2] |= (unsigned)*reinterpret_cast<const unsigned short *>(p + i) << (16 * (i & 1));
      }
    }
  }
  return out;
}

// Tiles of `tile` rows of stretches that begin at offsets[0 .. count] (ascending, offsets[0] = 0) and of one more
// up to `rows`: stretch e's tiles are numbered from offsets[e] / tile + e on. That leaves room for all of them,
// ceil(a) <= floor(a + b) - floor(b) + 1, so a tile's number alone says where it lies, without a list of tiles: the
// last e whose first number is not above it. Numbers run up to rows / tile + count; some have no rows.
__device__ __forceinline__ bool ragged_tile(const int *offsets, int count, int rows, int tile, int number, int &stretch,
                                            int &first, int &rows_here) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = count + 1;
  while (n > 1) {  // 64 places at a time
    const int step = (n + 63) / 64;
    const int e = lo + lane * step;
    const bool below = lane * step < n && offsets[e] / tile + e <= number;
    const int hits = __popcll(__ballot(below));
    const int skip = (hits - 1) * step;  // (lane 0 always hits)
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int begin = offsets[lo], end = lo == count ? rows : offsets[lo + 1];
  stretch = lo;
  const long long behind = (long long)(number - (begin / tile + lo)) * tile;  // of the stretch's first row
  if (behind >= end - begin) {
    first = end, rows_here = 0;
    return false;
  }
  first = begin + (int)behind;
  rows_here = end - first < tile ? end - first : tile;
  return true;
}
inline size_t ragged_tiles(int count, int rows, int tile) { return (size_t)(rows / tile) + count + 1; }

// A product over the rows of each expert may take them in parts of `part` rows, and experts that have more than that as
// sums of their parts' products, which lie in `sums` until they are added up. Parts are numbered as ragged tiles are;
// an expert without rows has one (of none). In any `part` rows, at most one part that is not its expert's first begins
// and at most one that is the first of several: where a part's sum lies follows from where it begins.
struct PartOfRows {
  int expert, first, rows;
  int sum;  // which of `sums`, or -1: the expert's only part
};
__device__ __forceinline__ bool part_of_rows(const int *offsets, int experts, int rows, int part, int number,
                                             PartOfRows &p) {
  const bool any = ragged_tile(offsets, experts, rows, part, number, p.expert, p.first, p.rows);
  if (p.expert == experts) return false;
  const int begin = offsets[p.expert], end = offsets[p.expert + 1];
  if (!any) {
    p.rows = 0, p.sum = -1;
    return begin == end && number == begin / part + p.expert;
  }
  p.sum = end - begin > part ? 2 * (p.first / part) + (p.first == begin) : -1;
  return true;
}

// launch(first block, blocks) until all of them are; a launch has at most 2^32 threads.
template <typename F>
inline int in_launches(size_t blocks, F launch) {
  constexpr size_t MOST = (size_t)1 << 22;
  if (blocks > UINT_MAX) return H2O4GPU_KMEANS_EARG;
  for (size_t b = 0; b < blocks; b += MOST) KM_TRY(launch((unsigned)b, (unsigned)(blocks - b < MOST ? blocks - b : MOST)));
  return H2O4GPU_KMEANS_OK;
}

// N values (of 4 or 8) side by side, at any address that a T may have: 2-byte ones that begin between words as one, the
// words behind it, and the last.
template <typename T, int N>
struct Beside {
  typedef T vector __attribute__((ext_vector_type(N)));
};
template <typename T, int N>
__device__ __forceinline__ void store_beside(T *to, typename Beside<T, N>::vector v) {
  constexpr int WORDS = N * (int)sizeof(T) / 4;
  typedef unsigned words __attribute__((ext_vector_type(WORDS)));
  struct __attribute__((packed, aligned(4))) Words {
    words v;
  };
  const words w = __builtin_bit_cast(words, v);
  if (sizeof(T) == 4 || !((size_t)to & 2)) {
    reinterpret_cast<Words *>(to)->v = w;
    return;
  }
  unsigned short *ends = reinterpret_cast<unsigned short *>(to);
  ends[0] = (unsigned short)w[0];
  unsigned *between = reinterpret_cast<unsigned *>(to + 1);
#pragma unroll
  for (int i = 0; i < WORDS - 1; ++i) between[i] = __builtin_amdgcn_alignbit(w[i + 1], w[i], 16);
  ends[N - 1] = (unsigned short)(w[WORDS - 1] >> 16);
}
template <typename T>
__device__ __forceinline__ void store_four(T *c, f32x4 v, int valid) {
  if (valid >= 4) {
    store_beside<T, 4>(c, typename Beside<T, 4>::vector{(T)v[0], (T)v[1], (T)v[2], (T)v[3]});
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < valid) c[j] = (T)v[j];
  }
}

}  // namespace kmhip
