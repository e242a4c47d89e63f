// Which kernel takes a product: rules on sizes, types, strides and addresses, on the host alone. C[m][n] is the sum over
// k of X[m][k] W[n][k]; of the matrices' gradient the rows are what is summed over, and m is C's first side, `k` here.
#pragma once

#include <limits.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>

namespace kmhip {

enum Kind { FORWARD, DROWS, DWEIGHTS };

// FEW_ROWS: thin_kernel, thin_columns_kernel; KEPT: kept_kernel; ANY_ROWS: product_kernel; TILES_128, TILES_256: pipe_kernel.
enum Way { FEW_ROWS, KEPT, ANY_ROWS, TILES_128, TILES_256 };

constexpr size_t BUFFER_BYTES = (size_t)1 << 32;  // what a buffer's offsets reach

// A product's operands. `size`: bytes of an element, 1 for microscaled 4-bit numbers; strides in elements.
struct ProductSizes {
  Kind kind;
  int size;
  const void *x, *w;
  size_t x_stride, w_stride, w_expert;
  int experts, rows, n, k;  // experts 0: one matrix and `rows` rows
  int part;                 // DWEIGHTS: rows of a part (rows_of_part)
};

// Whether a product is one of few rows: of an expert at most 16 (float32: 48) on average, beyond which tiles of 128 x 128
// are faster (27 experts of 5184 x 2504, 24 rows each: bfloat16 185 us against 199, 4 bits 63 against 68, float32 709
// against 423; 40 rows 193, 63 and 709 against 263, 99 and 566), or so few that the workgroups of 64 rows times 32 of the
// matrix are about as many as the CUs. Such tiles would be too few, and each has all of the columns: in one matrix of
// 2048 x 8192, 200 rows take 45 us here and 77 there, float16; 400 (432 workgroups) 89 and 77. In 4 bits and in float32 a
// tile's turn takes as long as three of these (4 bits, 400 rows 32 and 56 us, 800 60 and 55; float32 of 2048 x 4096, 400
// rows 114 and 244, 800 219 and 245). The average is what the host knows; the offsets lie on the GPU. Where one expert has
// most rows, its matrix is read for every 16 of them: 1024 rows of 64 experts of 4096 x 4096, bfloat16, take 549 us evenly
// shared (in tiles 372) and 473 all in one (52), in 4 bits 209 (138) and 182 (34). Matrices as large and as many as these, and
// those of few columns, would be faster in tiles from fewer rows on (8 rows each of the former 423 and 366, of 64 experts of
// 4096 x 1024 148 and 97), smaller and fewer ones not (of 8 experts of 2048 x 2048 20 and 26).
inline bool few_rows(int size, int rows, int experts, int n) {
  const int matrices = experts ? experts : 1;
  return rows / matrices <= (size == 4 ? 48 : 16) ||
         (rows / 64.0 + matrices / 2.0) * ((n + 31) / 32) <= (size == 2 ? 320 : 768);
}

// Whether some row of a matrix begins between words.
inline bool between_words(int size, const void *p, size_t stride) {
  return size == 2 && (((uintptr_t)p & 3) || (stride & 1));
}
// ... or of either operand. (Matrices of 4-byte elements begin at words however many elements they have, and of one matrix
// there is no next: 300 experts' 30000 rows of 255 with 513 x 255, float32, take 105 us in tiles and 125 as any rows, the rows'
// gradient 112 and 179.)
inline bool between_words(const ProductSizes &a) {
  return between_words(a.size, a.x, a.x_stride) || between_words(a.size, a.w, a.w_stride) ||
         (a.size == 2 && a.experts > 1 && (a.w_expert & 1));
}

// Rows of a part of a matrix's gradient. The tiles of all parts are to be two for each CU at most, an expert's last part
// taken to be half full; but no part has fewer than 512 rows, which take a tile some 10 us (float32 30), beside which a
// sum's way to memory and back is little. 2 experts' 100000 rows of 102 with 102, bfloat16, take 26 us in parts of 512
// rows, 30 of 1024 and 45 of 2048 (float32 56, 88, 163); 16 experts' 96000 of 256 with 256 59, 44 and 44. (For two tiles
// to a CU numbers are aimed at that the parts' unevenness leaves below 512: aimed at 512 themselves, that last case took
// 54 us.) Where the experts have as many tiles by themselves, parts are for one that has most of the rows. pipe_kernel
// shares its tiles out by their rows where there are none, so its parts have 4096 (float32 2048): 32 experts' 3200 rows of
// 1024 with 1024 take 37 us in parts of 1024 and 23 in none. Narrow matrices are product_kernel's, which does not:
// four tiles for each CU, and no fewer than 512 rows (1000 experts of 77 x 101 float32, 300 rows on average and one with
// 3794, take 130 us, in parts of 1024 156, of 2048 199; 16 experts' 64000 rows of 64 with 2048, in parts of 1024, 217, in
// one part an expert 325). A matrix of 128 tiles and more is in one part, which leaves CUs idle where few such have the rows:
// one expert's 65536 rows of 1024 with 2048, bfloat16, take 890 us, of 1024 with 1920 in parts 407; 64 experts' 65536 of 2048
// with 2048 530 us evenly shared, and 1930 where one expert has all of them. All parts' sums are at most 2 (1024 + 128) tiles of
// 64 KB.
inline int rows_of_part(int size, size_t rows, int experts, size_t out, size_t cols) {
  const size_t tiles = ((out + 127) / 128) * ((cols + 127) / 128);
  if (tiles >= 128) return INT_MAX;
  size_t part, least = 512;
  if (out < 128 || cols < 128)
    part = rows * tiles / 1024;
  else if (experts * tiles >= 512)
    part = rows * tiles / 512, least = size == 4 ? 2048 : 4096;
  else
    part = 2 * rows * tiles / (768 - experts * tiles);
  return (int)((part > least ? part : least) + 63) / 64 * 64;
}
inline size_t part_sums(int rows, int part) { return 2 * ((size_t)rows / part + 1); }
inline size_t sums_bytes(int size, size_t rows, int experts, size_t out, size_t cols) {
  const int part = rows_of_part(size, rows, experts, out, cols);
  return rows <= (size_t)part ? 0 : part_sums((int)rows, part) * out * cols * sizeof(float);
}

// Tiles of 256 x 256, or of 128 x 128, of which a CU holds two: by how often the card is filled with either (an expert's
// last tile is taken to be half full), and how long a stage then takes, 1.7 and 1.3 us. 64 experts' 65536 rows of 2048
// with 2048 x 2048 bfloat16 take 543 us in large tiles and 674 in small ones (both before the tiles were stored as they
// are now), 4 experts' 8000 rows of 1024 with 512 x 1024 27 and 16 us, 10 experts' 16941 rows of 4544 with 384 89 and 64,
// 160 experts' 49552 rows of 256 with 3392 188 and 191. float32 is bound by its matrix instructions: a small tile's stage
// takes 1.95 us for each that its CU has, a large one's 7.3, and what counts is how many a CU gets. In large and in small
// tiles take: 4 experts' 4096 rows of 2048 with 2048 x 2048 467 and 239 us (the rows' gradient 482 and 249), 8 experts'
// 6000 of 768 with 1536 186 and 145, 4 experts' 20000 of 640 with 640 158 and 166, 64 experts' 65536 of 1024 with 1024 951
// and 955; matrices' gradients 8 experts' 16384 of 512 with 2048 962 and 397, one expert's 4096 of 4096 with 4096 950 and 973. Of parts
// some numbers have no rows, and a CU may get two large tiles where another gets none, for the 6 % that they gain at best (8
// experts' 16384 rows of 1023 with 1025 968 and 627).
inline Way tiles_of(const ProductSizes &a) {
  auto turns = [&](int tile, int at_once) {
    const double n = (a.n + tile - 1) / tile;
    const double m = a.kind == DWEIGHTS ? (double)((a.k + tile - 1) / tile) *
                                              (a.part < a.rows ? a.rows / a.part + a.experts / 2 : a.experts)
                                        : (double)a.rows / tile + a.experts / 2.0;
    return ceil(m * n / at_once);
  };
  if (a.size == 4 && a.kind == DWEIGHTS && a.part < a.rows) return TILES_128;
  if (a.size == 4) return 7.3 * turns(256, 256) <= 1.95 * turns(128, 256) ? TILES_256 : TILES_128;
  return 1.7 * turns(256, 256) <= 1.3 * turns(128, 512) ? TILES_256 : TILES_128;
}

// A product of 16- or 32-bit numbers.
inline Way way_of(const ProductSizes &a) {
  const int each = a.rows / a.experts;
  // few rows of an expert, see few_rows (the rows' gradient: 8 experts of 4096 x 4096, 24 rows each, bfloat16, 46 us there
  // and 54 in tiles, but 300 experts of 512 x 512, 20 rows each, 50 and 32; float32 of the first with 48 rows each 173 and
  // 262, of 300 experts with 50 rows each 173 and 176); far: an offset of a tile's last row would not fit a buffer
  const bool far = a.x_stride * a.size >= BUFFER_BYTES / 512 || a.w_stride * a.size >= BUFFER_BYTES / 512;
  const bool few = a.kind == FORWARD ? few_rows(a.size, a.rows, a.experts, a.n) : each <= (a.size == 4 ? 64 : 16);
  if (a.kind != DWEIGHTS && (far || few)) return FEW_ROWS;
  // Tiles that a matrix does not fill cost float32 and the matrices' gradient their products, which product_kernel leaves
  // out (16 experts' 64000 rows of 2048 with 64 x 2048, float32, 181 us there and 246 here, the gradient 222 and 347);
  // other products wait for memory (64 experts' 64000 rows of 640 with 16 x 640, bfloat16, 31 and 18). float32 gradients of
  // few rows are faster there (8 experts' of 4096 x 4096, 24 rows each, 163 and 195, 48 rows each 225 and 196; bfloat16 86
  // and 68, 88 and 67).
  const int least = a.size == 4 || a.kind == DWEIGHTS ? 128 : 16;
  if (!between_words(a) && a.n >= least && (a.kind != DWEIGHTS || (a.k >= least && (a.size == 2 || each >= 32))))
    return tiles_of(a);
  return ANY_ROWS;
}

// A product of microscaled 4-bit numbers in rows of `pitch` bytes. x_rows: rows of x, which are gathered if `gather`.
inline Way way_of_four(int rows, int experts, int out, size_t cols, size_t pitch, bool gather, size_t x_rows) {
  // what a buffer's offsets reach: the gathered x in all, 256 rows of a matrix
  const bool reached = (!gather || x_rows * pitch < BUFFER_BYTES) && pitch < BUFFER_BYTES / 512;
  // x of 17 to 64 rows is kept where its columns fit the registers, however few rows the matrix has (33 rows of 8192 times 256
  // 9.0 us and 12.3 as few rows, 64 rows of 1024 times 4000 6.6 and 10.2, 17 rows of 4096 times 2048 6.7 and 6.6, from Python)
  if (!reached || few_rows(1, rows, experts, out))
    return !experts && rows > 16 && rows <= 64 && cols <= 8192 ? KEPT : FEW_ROWS;
  return tiles_of(ProductSizes{FORWARD, 1, nullptr, nullptr, 0, 0, 0, experts, rows, out, 0, 0});
}

}  // namespace kmhip
