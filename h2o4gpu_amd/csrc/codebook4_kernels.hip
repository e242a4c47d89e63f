// Matrices of 4-bit codes: compressing one, and its product with tokens, alone or a matrix per expert.
#include "experts_common.h"
#include "mfma_traits.h"

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
  const int groups = (cols + group - 1) / group;
  for (int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); n < out; n += (int64_t)gridDim.x * 4) {
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

// A matrix (or one per expert) in the order the product reads it, see launch_layout4.
struct Matrix4 {
  const uint4 *codes = nullptr;
  const void *scales = nullptr;
  const void *books = nullptr;
  int64_t book_stride = 0;
  int64_t out = 0;
  int cols = 0;
  int per = 1;  // scales of a row for 128 columns
};

// The product on the matrix cores. x is the "A" operand (rows of the result tile: 16 tokens), the
// matrix the "B" operand (columns: 16 of y), so a lane holds one column of y and every scale it
// applies is its own column's:
//   A[i = lane % 16][k = VK * (lane / 16) + 0 .. VK-1], B[k likewise][j = lane % 16],
//   accumulator v: D[i = 4 * (lane / 16) + v][j = lane % 16].
// The matrix lies in tiles of 16 rows and 128 columns, each the 1024 bytes that a wavefront loads at once:
// lane (r, q) has 8 columns of each 32 of row r, so that no instruction mixes columns of two scales,
// and a wavefront that goes along its columns reads one stretch of memory. (Read from rows as they
// are, 64 bytes of 16 rows at a time and 2 bytes of 16 rows of scales, 8192 x 8192 takes 16 us at one
// token.) Codes become values through a table of pairs in LDS, indexed by a whole byte: 256
// entries of 256 bytes, each with a copy of the pair for every bank, so that reads do not collide and an
// address is one byte permutation (a table in registers takes 3.1 vector instructions a code, this one
// half an instruction and half a read). Products of 16-bit values are exact in float, sums are float; the
// scale is applied to the sum over its group.
template <typename T>
struct Mfma4;

template <>
struct Mfma4<bfloat16_t> {
  typedef bfloat16_t vec __attribute__((ext_vector_type(8)));
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
  static __device__ __forceinline__ floatx4 mma(const unsigned *a, const unsigned *b, floatx4 c) {
    vec va, vb;
    __builtin_memcpy(&va, a, 16);
    __builtin_memcpy(&vb, b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(va, vb, c, 0, 0, 0);
  }
};

template <>
struct Mfma4<float> {
  static __device__ __forceinline__ floatx4 mma(const unsigned *a, const unsigned *b, floatx4 c) {
#pragma unroll
    for (int i = 0; i < 8; i++)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
};

static const int TABLE_BYTES = 256 * 256;

// The same bytes at an address that is only aligned to its elements.
typedef unsigned uintx4_u __attribute__((ext_vector_type(4), aligned(2)));

// 8 values of x as 32-bit words.
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
// (left: columns from `at` to the row's end, negative behind it; at[left - 1] is the row's last)
template <typename T>
__device__ __forceinline__ void load_x8_end(const T *at, int left, unsigned (&w)[2 * sizeof(T)]) {
  if (left >= 8) {
    load_x8<T>(at, w);
    return;
  }
  // (as if new here: 32 offsets made ahead of the loops would take the registers of the loops)
  asm volatile("" : "+v"(left));
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = at[i < left ? i : left - 1];  // every load on its way before the first is used
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = i < left ? v[i] : (T)0.f;
  __builtin_memcpy(w, v, sizeof(v));
}

// 8 codes as 8 values: byte b of the word names a pair, whose copy for this lane lies lane_at into the entry.
// The table is the first thing in LDS (address 0): an address that had to be added to would cost as much as
// the permutation that makes it.
template <typename T>
__device__ __forceinline__ void decode8(unsigned word, unsigned lane_at,
                                        unsigned (&w)[2 * sizeof(T)]) {
  typedef unsigned Two __attribute__((ext_vector_type(2)));
  typedef typename std::conditional<sizeof(T) == 4, Two, unsigned>::type Pair;
  typedef const __attribute__((address_space(3))) Pair *LdsPair;
  // address = 256 * byte + lane_at: result bytes 0, 0, word's byte b, lane_at's byte 0
  const unsigned at[4] = {__builtin_amdgcn_perm(word, lane_at, 0x0c0c0400), __builtin_amdgcn_perm(word, lane_at, 0x0c0c0500),
                          __builtin_amdgcn_perm(word, lane_at, 0x0c0c0600), __builtin_amdgcn_perm(word, lane_at, 0x0c0c0700)};
  Pair p[4];
#pragma unroll
  for (int b = 0; b < 4; b++) p[b] = *reinterpret_cast<LdsPair>((uint32_t)at[b]);
  __builtin_memcpy(w, p, sizeof(p));
}

struct Product4Args {
  Matrix4 m;
  RowSource src;
  int64_t xs, ys;
  int splits;  // wavefronts that share a tile's columns
};

// A workgroup's expert and rows of y; hi <= lo where it has none.
struct Share {
  int expert = 0;
  int64_t lo = 0, hi = 0;
};

// With experts, blockIdx.y is one, or, where there are fewer rows than experts, a row: the workgroups of an
// expert's first row then have all of its rows. The last blockIdx.y writes zeros to the rows that have none.
template <typename T>
__device__ __forceinline__ Share share_of(const Product4Args &a, int *found, T *y) {
  Share s;
  s.hi = a.src.rows;
  if (!a.src.offsets) return s;
  const int E = a.src.experts;
  if (blockIdx.y == gridDim.y - 1) {
    for (int64_t p = a.src.offsets[E] + blockIdx.z * gridDim.x + blockIdx.x; p < s.hi; p += gridDim.x * gridDim.z)
      for (int64_t n = threadIdx.x; n < a.m.out; n += blockDim.x) y[p * a.ys + n] = (T)0.f;
    s.hi = 0;
    return s;
  }
  if ((int)gridDim.y - 1 == E) {
    s.expert = blockIdx.y;
    s.lo = a.src.offsets[s.expert];
    s.hi = a.src.offsets[s.expert + 1];
    return s;
  }
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
  s.expert = __builtin_amdgcn_readfirstlane(found[0]);
  s.lo = p;
  s.hi = s.expert >= 0 ? __builtin_amdgcn_readfirstlane(found[1]) : p;
  __syncthreads();
  return s;
}

// Where row p of y has its x.
template <typename T>
__device__ __forceinline__ const T *x_row(const T *x, const Product4Args &a, int64_t p) {
  return x + (a.src.order ? (int64_t)((unsigned)a.src.order[p] / (unsigned)a.src.top_k) : p) * a.xs;
}

// The pair table of an expert's codebook: 16 lanes write an entry, a wavefront four in a row, so that no two
// lanes write to one bank.
template <typename T>
__device__ __forceinline__ void make_table(char *lds, const Matrix4 &m, int e) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, r = lane & 15;
  const float held = (float)static_cast<const T *>(m.books)[e * m.book_stride + r];
  for (int byte = wave * 4 + (lane >> 4); byte < 256; byte += waves * 4) {
    const T low = (T)__shfl(held, byte & 15, 64), high = (T)__shfl(held, byte >> 4, 64);
    T pair[16 / sizeof(T)];
#pragma unroll
    for (int c = 0; c < (int)(16 / sizeof(T)); c += 2) {
      pair[c] = low;
      pair[c + 1] = high;
    }
    uint4 four;
    __builtin_memcpy(&four, pair, 16);
    *reinterpret_cast<uint4 *>(lds + byte * 256 + r * 16) = four;
  }
  __syncthreads();
}

// The 128 columns of NT tiles, on their way to or in registers: scales as they lie in memory, so that nothing
// waits for them before they are used.
template <typename S, int NT, int PER>
struct Tiles {
  struct alignas(sizeof(S) * PER) Scales {
    S v[PER];
  };
  uint4 words[NT];
  Scales scale[NT];
};

// A wavefront's place in the matrix.
template <typename S, int NT, int PER>
struct Reader {
  typedef Tiles<S, NT, PER> Held;
  const uint4 *codes;
  const typename Held::Scales *scales;
  int64_t at[NT];

  __device__ __forceinline__ Reader(const Matrix4 &m, int e, int tiles16, int subs) {
    codes = m.codes + (int64_t)e * tiles16 * subs * 64 + (threadIdx.x & 63);
    scales = static_cast<const typename Held::Scales *>(m.scales) + (int64_t)e * tiles16 * subs * 16 +
             (threadIdx.x & 15);
  }
  __device__ __forceinline__ void move_to(int tile, int tiles16, int subs) {  // (behind the last tile: the last again)
#pragma unroll
    for (int t = 0; t < NT; t++) at[t] = (int64_t)(tile + t < tiles16 ? tile + t : tiles16 - 1) * subs;
  }
  __device__ __forceinline__ void fetch(Held &h, int sub) const {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      h.words[t] = codes[(at[t] + sub) * 64];
      h.scale[t] = scales[(at[t] + sub) * 16];
    }
  }
};

// One tile's 128 columns as values: 4 operands of a product. Every table read is on its way before what follows.
template <typename T>
__device__ __forceinline__ void decode(const uint4 &words, unsigned lane_at, unsigned (&b)[4][2 * sizeof(T)]) {
  const unsigned d[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
  for (int i = 0; i < 4; i++) decode8<T>(d[i], lane_at, b[i]);
  __builtin_amdgcn_sched_barrier(0);
}

// Both kernels: a workgroup's wavefronts have blockDim / 64 / splits tiles of 16 * NT columns of y at a time;
// `splits` wavefronts share a tile's columns of the matrix, each a stretch of them, 128 at a time with the
// next R on their way, and add their sums up in LDS. PER: scales of a row for 128 columns (1, 2 or 4).

// Up to MP rows of y at a time (1 or 4). A product's 16 rows of x are these rows in G = 16 / MP pieces of 128
// columns, loaded once for G tiles of the matrix: the result's row p * MP + m is y's row m with piece p, and of
// each product only the rows of the tile's own piece are kept. Loading the matrix bounds it: 1 x 8192 x 8192 takes
// 10.4 us (14.3 with a row of x in each of the 16; 9 to 10 for loading the tiles and nothing else), 1 x 4096 x 4096
// 5.8 (5.0; an empty launch 2.5), 4 x 8192 x 8192 12.5, 1 x 32768 x 8192 31, which is 4.4 TB/s (26).
template <typename T, typename S, int MP, int PER>
__global__ __launch_bounds__(512, sizeof(T) == 2 ? 4 : 2) void product4_few_kernel(const T *x, T *y, Product4Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int G = 16 / MP, SETS = MP == 4 ? 2 : 1;
  constexpr int R = MP == 4 && PER > 1 ? 2 : 4;  // (as many as there are registers for)
  typedef unsigned Frag[4][2 * sizeof(T)];
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  float *red = reinterpret_cast<float *>(lds + TABLE_BYTES);
  const int teams = waves / a.splits, team = wave / a.splits, part = wave % a.splits;
  const int tiles16 = (int)((a.m.out + 15) >> 4), subs = (a.m.cols + 127) >> 7;
  const Share share = share_of(a, reinterpret_cast<int *>(red), y);
  const int64_t begin = share.lo + (int64_t)blockIdx.z * MP, hi = share.hi;
  if (begin >= hi) return;
  const unsigned lane_at = (lane * 2 * sizeof(T)) & 255;
  const int cols = a.m.cols, full = cols >> 7;
  const int first = full * part / a.splits, count = full * (part + 1) / a.splits - first;
  Reader<S, 1, PER> reader(a.m, share.expert, tiles16, subs);

  bool have_table = false;
  for (int tile0 = blockIdx.x * teams; tile0 < tiles16; tile0 += gridDim.x * teams) {
    const int tile = tile0 + team;
    const bool mine = tile < tiles16;
    reader.move_to(tile, tiles16, subs);
    for (int64_t lo = begin; lo < hi; lo += (int64_t)gridDim.z * MP) {
      const T *row = x_row(x, a, lo + r % MP < hi ? lo + r % MP : hi - 1) + 8 * q;
      const auto load_x = [&](Frag &xf, int b) {  // (pieces behind the last tile: the last tile's again)
        const int64_t at = (int64_t)(first + (b + r / MP < count ? b + r / MP : count - 1)) * 128;
#pragma unroll
        for (int i = 0; i < 4; i++) load_x8<T>(row + (at + 32 * i), xf[i]);
      };
      float acc[MP] = {};  // over the pieces of lanes q
      // j: the piece, of which the last two bits are known when this is compiled
      const auto multiply = [&](const Frag &xf, const Tiles<S, 1, PER> &h, int j, int piece) {
        Frag bf;
        decode<T>(h.words[0], lane_at, bf);
        const bool own = q == piece * MP / 4;
        floatx4 sum = {};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          sum = Mfma4<T>::mma(xf[i], bf[i], sum);
          if ((i + 1) % (4 / PER) == 0) {
            const float by = (float)h.scale[0].v[i * PER / 4];
#pragma unroll
            for (int m = 0; m < MP; m++) acc[m] = own ? fmaf(by, sum[(MP * j + m) & 3], acc[m]) : acc[m];
            sum = floatx4{0.f, 0.f, 0.f, 0.f};
          }
        }
      };
      Tiles<S, 1, PER> held[R];
      Frag xf[SETS];
      if (mine && count > 0) {
        load_x(xf[0], 0);
#pragma unroll
        for (int j = 0; j < R; j++)
          if (j < count) reader.fetch(held[j], first + j);
      }
      if (!have_table) make_table<T>(lds, a.m, share.expert);
      have_table = true;
      if (mine) {
        const auto four = [&](const Frag &now, int b) {
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (b + j >= count) break;
            multiply(now, held[j % R], j, (b + j) % G);
            if (b + j + R < count) reader.fetch(held[j % R], first + b + j + R);
          }
        };
        if (SETS == 1) {
          for (int b = 0; b < count; b += 4) {
            if (b > 0 && b % G == 0) load_x(xf[0], b);
            four(xf[0], b);
          }
        } else {  // a set of x lasts for four tiles: the next is on its way meanwhile
          for (int b = 0; b < count; b += 8) {
            if (b + 4 < count) load_x(xf[SETS - 1], b + 4);
            four(xf[0], b);
            if (b + 4 >= count) break;
            if (b + 8 < count) load_x(xf[0], b + 8);
            four(xf[SETS - 1], b + 4);
          }
        }
        if ((cols & 127) && part == 0) {  // the columns behind the last whole 128 (part 0 has the fewest before)
          reader.fetch(held[0], full);
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int k = full * 128 + 32 * i;
            load_x8_end<T>(row + k, cols - k - 8 * q, xf[0][i]);
          }
          multiply(xf[0], held[0], 0, 0);
        }
      }
      // the four lanes of a column and the wavefronts of a tile, in their order
      const int tokens = hi - lo < MP ? (int)(hi - lo) : MP;
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MP; m++) red[(wave * MP + m) * 64 + lane] = acc[m];
      __syncthreads();
      for (int i = lane + 64 * part; mine && i < tokens * 16; i += 64 * a.splits) {
        const int m = i >> 4, c = i & 15;
        const int64_t n = 16 * (int64_t)tile + c;
        if (n < a.m.out) {
          const float *from = red + (team * a.splits * MP + m) * 64 + c;
          float sum = 0.f;
          for (int w = 0; w < a.splits; w++, from += MP * 64) sum += (from[0] + from[16]) + (from[32] + from[48]);
          y[(lo + m) * a.ys + n] = (T)sum;
        }
      }
    }
  }
}

// 16 * MT rows of y at a time, a row of x in each of a product's 16. Rows of x behind the last one are read from
// the last: their results are not written.
// A product wants 8 columns of 16 different rows from 16 neighbouring lanes. x is not loaded like that: 16 lanes load
// 128 columns of one row, and a wavefront's own 16 x 128 corner of LDS turns them (33 x 8192 x 8192: 25.4 -> 21.8
// us). Piece c of row r lies at place c ^ r of its row there, so that 16 rows' pieces c lie in different banks.
// What bounds it at that size: every workgroup reads all of x, from L2; without these loads 16.5 us, with the loads
// and without the turn 20.1, and a step's x on its way a step earlier 21.7. 16 x 8192 x 8192: 14.6 us, 64: 23.7.
template <typename T, typename S, int MT, int NT, int R, int PER>
__global__ __launch_bounds__(512) void product4_kernel(const T *x, T *y, Product4Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int W = 2 * sizeof(T), SZ = 8 * sizeof(T);  // words and bytes of a piece: 8 values
  typedef unsigned Piece __attribute__((ext_vector_type(W)));
  typedef unsigned Piece_u __attribute__((ext_vector_type(W), aligned(sizeof(T))));
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  char *turn = lds + TABLE_BYTES + wave * (256 * SZ);
  float *red = reinterpret_cast<float *>(lds + TABLE_BYTES);  // (in the same place, when the corners are done with)
  const int teams = waves / a.splits, team = wave / a.splits, part = wave % a.splits;
  const int tiles16 = (int)((a.m.out + 15) >> 4), subs = (a.m.cols + 127) >> 7;
  const Share share = share_of(a, reinterpret_cast<int *>(red), y);
  const int64_t begin = share.lo + (int64_t)blockIdx.z * (16 * MT), hi = share.hi;
  if (begin >= hi) return;
  const unsigned lane_at = (lane * 2 * sizeof(T)) & 255;
  const int cols = a.m.cols, full = cols >> 7;
  const int first = full * part / a.splits, count = full * (part + 1) / a.splits - first;
  Reader<S, NT, PER> reader(a.m, share.expert, tiles16, subs);

  bool have_table = false;
  for (int tile0 = blockIdx.x * teams; tile0 * NT < tiles16; tile0 += gridDim.x * teams) {
    const int tile = (tile0 + team) * NT;
    const bool mine = tile < tiles16;
    reader.move_to(tile, tiles16, subs);
    for (int64_t lo = begin; lo < hi; lo += (int64_t)gridDim.z * (16 * MT)) {
      // load j of 16 rows: row 4 j + q, its piece r ^ (4 j + q)
      const T *from[MT][4];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int64_t p = lo + 16 * m + 4 * j + q;
          from[m][j] = x_row(x, a, p < hi ? p : hi - 1) + 8 * (r ^ (4 * j + q));
        }
      floatx4 acc[MT][NT] = {};
      Tiles<S, NT, PER> held[R];
      Piece raw[R][MT][4];
      const auto fetch = [&](int k, int sub) {
        reader.fetch(held[k], sub);
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int j = 0; j < 4; j++) raw[k][m][j] = *reinterpret_cast<const Piece_u *>(from[m][j] + (int64_t)sub * 128);
      };
      unsigned xf[MT][4][W];
      const auto turn_x = [&](int k) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
#pragma unroll
          for (int j = 0; j < 4; j++) *reinterpret_cast<Piece *>(turn + (64 * j + lane) * SZ) = raw[k][m][j];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const Piece v = *reinterpret_cast<const Piece *>(turn + (16 * r + ((4 * i + q) ^ r)) * SZ);
            __builtin_memcpy(xf[m][i], &v, SZ);
          }
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
      };
      const auto multiply = [&](const Tiles<S, NT, PER> &h, int t) {
        unsigned b[4][W];
        decode<T>(h.words[t], lane_at, b);
        floatx4 sum[MT] = {};
#pragma unroll
        for (int i = 0; i < 4; i++) {
#pragma unroll
          for (int m = 0; m < MT; m++) {
            sum[m] = Mfma4<T>::mma(xf[m][i], b[i], sum[m]);
            if ((i + 1) % (4 / PER) == 0) {
              const float sc = (float)h.scale[t].v[i * PER / 4];
#pragma unroll
              for (int v = 0; v < 4; v++) acc[m][t][v] = fmaf(sc, sum[m][v], acc[m][t][v]);
              sum[m] = floatx4{0.f, 0.f, 0.f, 0.f};
            }
          }
        }
      };
      if (mine) {
#pragma unroll
        for (int k = 0; k < R; k++)
          if (k < count) fetch(k, first + k);
      }
      if (!have_table) make_table<T>(lds, a.m, share.expert);
      have_table = true;
      if (mine) {
        for (int b = 0; b < count; b += R) {
#pragma unroll
          for (int k = 0; k < R; k++) {
            if (b + k >= count) break;
            turn_x(k);
#pragma unroll
            for (int n = 0; n < NT; n++) multiply(held[k], n);
            if (b + R + k < count) fetch(k, first + b + R + k);
          }
        }
        if ((cols & 127) && part == 0) {  // the columns behind the last whole 128 (part 0 has the fewest before)
          reader.fetch(held[0], full);
#pragma unroll
          for (int m = 0; m < MT; m++) {
            const T *row = x_row(x, a, lo + 16 * m + r < hi ? lo + 16 * m + r : hi - 1) + 8 * q;
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const int k = full * 128 + 32 * i;
              load_x8_end<T>(row + k, cols - k - 8 * q, xf[m][i]);
            }
          }
#pragma unroll
          for (int t = 0; t < NT; t++) multiply(held[0], t);
        }
      }
      // the sums of a tile's wavefronts, in their order
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const int tokens = hi - lo - 16 * m < 16 ? (int)(hi - lo - 16 * m) : 16;
        if (tokens <= 0) break;
        if (a.splits == 1) {
          if (mine) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
              for (int v = 0; v < 4; v++) {
                const int64_t n = 16 * (int64_t)(tile + t) + r;
                if (4 * q + v < tokens && n < a.m.out) y[(lo + 16 * m + 4 * q + v) * a.ys + n] = (T)acc[m][t][v];
              }
          }
          continue;
        }
        __syncthreads();
        if (4 * q < tokens) {
#pragma unroll
          for (int t = 0; t < NT; t++)
#pragma unroll
            for (int v = 0; v < 4; v++) red[(wave * (4 * NT) + 4 * t + v) * 64 + lane] = acc[m][t][v];
        }
        __syncthreads();
        // (token, column): 16 neighbours write 16 columns of one row
        for (int i = lane + 64 * part; mine && i < tokens * 16 * NT; i += 64 * a.splits) {
          const int token = i / (16 * NT), c = i % (16 * NT);
          const int64_t n = 16 * (int64_t)tile + c;
          if (n < a.m.out) {
            const float *at = red + team * a.splits * (4 * NT * 64) + (4 * (c >> 4) + (token & 3)) * 64 +
                              (token >> 2) * 16 + (c & 15);
            float total = 0.f;
            for (int w = 0; w < a.splits; w++) total += at[w * (4 * NT * 64)];
            y[(lo + 16 * m + token) * a.ys + n] = (T)total;
          }
        }
      }
      if (a.splits > 1) __syncthreads();  // (before the corners are used again)
    }
  }
}

// ---------------------------------------------------------------------------
// the order the product reads a matrix in
// ---------------------------------------------------------------------------

// Tile (row / 16, column / 128), lane (r, q): 16 bytes whose word i holds row r's columns 32 i + 8 q .. + 7
// of the tile. Scales: a tile's 16 rows, one each, or four each (one per 32 columns) where a group ends
// within 128. Rows and columns behind the matrix have code 0 and scale 0.
__global__ __launch_bounds__(256) void layout4_codes_kernel(const uint8_t *codes, int64_t pitch, int64_t out, int cols,
                                                            int64_t tiles16, int subs, int64_t lanes, uint4 *to) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < lanes; i += (int64_t)gridDim.x * 256) {
    const int lane = i & 63, r = lane & 15, q = lane >> 4;
    const int sub = (i >> 6) % subs;
    const int64_t tile = (i >> 6) / subs, e = tile / tiles16, n = (tile % tiles16) * 16 + r;
    const uint8_t *row = codes + (e * out + n) * pitch;
    unsigned w[4] = {0, 0, 0, 0};
    if (n < out) {
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int k0 = sub * 128 + 32 * j + 8 * q;
        if (k0 + 8 <= cols) {
          __builtin_memcpy(&w[j], row + k0 / 2, 4);
        } else {
          for (int b = 0; b < 4 && k0 + 2 * b < cols; b++)
            w[j] |= (row[k0 / 2 + b] & (k0 + 2 * b + 1 < cols ? 255u : 15u)) << (8 * b);
        }
      }
    }
    to[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename S>
__global__ __launch_bounds__(256) void layout4_scales_kernel(const S *scales, int64_t out, int groups, int group,
                                                             int64_t tiles16, int subs, int per, int64_t count,
                                                             S *to) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    const int p = i % per, r = (i / per) & 15;
    const int64_t t = i / per / 16, tile = t / subs, e = tile / tiles16, n = (tile % tiles16) * 16 + r;
    const int g = ((t % subs) * 128 + p * (128 / per)) / group;
    to[i] = n < out && g < groups ? scales[(e * out + n) * groups + g] : (S)0;
  }
}

static const size_t MOST_OUT = 1 << 24, MOST_COLS4 = 1000000, MOST_ROWS4 = 2147483646;

static bool sizes_ok(size_t experts, size_t out, size_t cols, int group) {
  return experts >= 1 && experts <= H2O4GPU_EXPERTS_MAX_EXPERTS && out >= 1 && out <= MOST_OUT && cols >= 1 &&
         cols <= MOST_COLS4 && group >= 32 && group % 32 == 0 && group <= H2O4GPU_CODEBOOK4_MAX_GROUP;
}

static bool strided_ok(int dtype, const void *p, size_t stride, size_t cols) {
  return p && aligned_to(p, type_size(dtype)) && stride >= cols && stride <= ((size_t)1 << 40);
}

// Rows of codes and scales as quantize writes them.
static bool packed_ok(const void *codes, size_t pitch, size_t cols, int scale_dtype, const void *scales) {
  return codes && pitch >= (cols + 1) / 2 && pitch <= ((size_t)1 << 32) && known_type(scale_dtype) && scales &&
         aligned_to(scales, type_size(scale_dtype));
}

static size_t tiles_of(size_t out) { return (out + 15) / 16; }
static size_t subs_of(size_t cols) { return (cols + 127) / 128; }
static int scales_per_sub(int group) { return group % 128 == 0 ? 1 : group % 64 == 0 ? 2 : 4; }
static unsigned blocks_for(size_t items) { return (unsigned)((items + 255) / 256 < 65536 ? (items + 255) / 256 : 65536); }

// rows: of y that a workgroup has at a time, tile: columns of y a team of wavefronts has, share_rows: rows of y
// that a matrix has, about.
template <typename T>
static int launch_product4(void (*kernel)(const T *, T *, Product4Args), int rows, int tile, const T *x, T *y,
                           Product4Args a, int64_t share_rows, int waves, int splits, hipStream_t s) {
  const size_t sums = (size_t)waves * 64 * (tile / 16) * (rows < 4 ? rows : 4) * sizeof(float);
  const size_t corners = rows >= 16 ? (size_t)waves * 256 * 8 * sizeof(T) : 0;
  const size_t lds = TABLE_BYTES + (sums > corners ? sums : corners);
  KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds));
  a.splits = splits;
  const int teams = waves / splits;
  const unsigned tiles = (unsigned)((a.m.out + tile - 1) / tile);
  unsigned gx = (tiles + teams - 1) / teams;
  const unsigned gy = a.src.offsets ? (unsigned)(a.src.rows < a.src.experts ? a.src.rows : a.src.experts) + 1 : 1;
  const int64_t steps = (share_rows + rows - 1) / rows;
  const unsigned gz = (unsigned)(steps < 256 ? steps : 256);
  // no more workgroups than run at once, twice over: one that has several tiles makes its table once
  const unsigned most = 1024 / (gy * gz) > 0 ? 1024 / (gy * gz) : 1;
  if (gx > most) gx = most;
  hipLaunchKernelGGL(kernel, dim3(gx, gy, gz), dim3(64 * waves), lds, s, x, y, a);
  return launched();
}

// Rows of y that a workgroup has at a time and columns that a team of its eight wavefronts has, both in 16s, and
// the wavefronts of a team, which share the columns of the matrix.
struct Tiling4 {
  int mt, nt, splits;
};

// As few wavefronts to a team as give every CU two workgroups (of `all` tiles of 16 x 16 * mt).
static Tiling4 with_splits(int mt, int nt, int64_t all, int subs) {
  int splits = 8;
  while (splits > 1 && (splits / 2 >= subs || (all + nt - 1) / nt * (splits / 2) >= 4096)) splits /= 2;
  return Tiling4{mt, nt, splits};
}

// Many experts, whose rows are not known here: with this many tiles, counting turns by their average is worse (64
// experts of 2048 x 4096 with four rows each: 84 us; with 32 rows 206 against 190; 16 of 3000 x 3000 in float with
// six rows 74 against 67), with fewer it is better (8 experts of 3000 x 4096 with four rows: 18 against 26, with 32
// rows 35 against 44). x is read once for every 16 * nt columns of y and a matrix once for every 16 * mt rows, so both
// are as large as there are registers for (a float takes twice as many, and so do four scales for 128 columns).
// 64 experts of 2048 x 4096 with four rows each: 59 us with 1 x 4, 97 with 1 x 2.
static Tiling4 experts_tiling(int64_t rows, int64_t tiles, int subs, int per, bool two_bytes) {
  if (rows <= 16) return with_splits(1, two_bytes && per < 4 ? 4 : 2, tiles, subs);
  // (640 tokens, four choices: 224 us with 2 x 4, 244 with 3 x 2; groups of 64: 246 with 2 x 3, 227 with 3 x 2)
  if (two_bytes && per == 2 && rows > 32 && rows <= 48) return with_splits(3, 2, tiles, subs);
  return with_splits(2, !two_bytes ? 1 : per == 1 ? 4 : per == 2 ? 3 : 2, tiles, subs);
}

// A matrix, or a few: the least of what was found to describe the kernel's time, workgroups on 256 CUs in turns (a
// CU has registers for one), each with a start and an end that take as long as 20 steps of 1 x 1, and a step of 128
// columns that takes one more for every tile and two for every 16 rows after the first. 8192 columns: 16 rows x 8192 take
// 14.6 us with 1 x 2, 16.1 with 1 x 3, 18.5 with 1 x 4; x 11000, 24.9, 16.8 and 19.9. 33 rows x 8192: 21.6 with
// 3 x 2, 29.9 with 2 x 2; x 11008, 38.1 with 3 x 2 and 32.8 with 2 x 3 and half the teams.
static Tiling4 product_tiling(int64_t rows, int64_t tiles, int64_t shares, int subs, int per, bool two_bytes) {
  // mt, nt, and for how many scales of 128 columns there are registers. (Two float scales beside 16-bit rows are more
  // than there is room for with 3 x 2 and 1 x 4, by 12 and 24 bytes a lane: 48 rows x 8192 x 8192, groups of 64, take 23.2
  // us so and 22.0 with scales of 16 bits, of which 6 % fewer bytes are loaded; 64 experts of 2048 x 4096 with four
  // rows each 76 and 74.)
  static const int halves[][3] = {{3, 2, 2}, {2, 4, 1}, {2, 3, 2}, {1, 4, 2},
                                  {1, 3, 4}, {2, 2, 4}, {1, 2, 4}, {1, 1, 4}};
  static const int floats[][3] = {{2, 1, 4}, {1, 2, 4}, {1, 1, 4}};
  Tiling4 best{1, 1, 8};
  int64_t least = INT64_MAX;
  for (int i = 0; i < (two_bytes ? 8 : 3); i++) {
    const int *shape = two_bytes ? halves[i] : floats[i];
    const int mt = shape[0], nt = shape[1];
    if (per > shape[2] || (mt > 1 && rows <= 16 * (mt - 1))) continue;
    const int64_t steps = (rows + 16 * mt - 1) / (16 * mt), wide = (tiles + nt - 1) / nt;
    for (int splits = 8; splits >= 1; splits /= 2) {
      if (splits > 1 && splits / 2 >= subs) continue;
      const int64_t turns = ((wide + 8 / splits - 1) / (8 / splits) * steps * shares + 255) / 256;
      const int64_t time = turns * (20 + (int64_t)((subs + splits - 1) / splits) * (nt + 2 * (mt - 1)));
      if (time < least) {
        least = time;
        best = Tiling4{mt, nt, splits};
      }
    }
  }
  return best;
}

static int product4(int dtype, const void *x, size_t x_stride, const Matrix4 &m, int scale_dtype,
                    const RowSource &src, void *y, size_t y_stride, hipStream_t s) {
  Product4Args a;
  a.m = m;
  a.src = src;
  a.xs = (int64_t)x_stride;
  a.ys = (int64_t)y_stride;
  const int subs = (int)subs_of(m.cols);
  const int64_t tiles = (int64_t)tiles_of(m.out);
  // rows that a matrix has, about, and matrices (or workgroups for a row each)
  const int64_t shares = !src.offsets ? 1 : src.rows < src.experts ? src.rows : src.experts;
  const int64_t rows = (src.rows + shares - 1) / shares;
  const bool two_bytes = dtype != H2O4GPU_EXPERTS_FLOAT32;
  // Few rows: the kernel that loads x least. Experts' rows are not spread evenly, and where there are tiles for
  // every wavefront wide ones are better still (64 experts of 2048 x 4096, 128 rows: 53 us against 82; 16 rows: 18
  // against 15).
  const bool few = src.rows == 1 || (src.offsets ? rows <= 2 && tiles * shares < 4096 : rows <= 4);
  const Tiling4 t = few ? with_splits(1, 1, tiles * shares, subs)
                    : src.offsets && tiles * shares >= (two_bytes ? 4096 : 1024)
                        ? experts_tiling(rows, tiles * shares, subs, m.per, two_bytes)
                        : product_tiling(rows, tiles, shares, subs, m.per, two_bytes);
  const int waves = 8, mt = t.mt, nt = t.nt, splits = t.splits;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    const T *tx = static_cast<const T *>(x);
    T *ty = static_cast<T *>(y);
    return with_type(scale_dtype, [&](auto stag) {
      typedef typename decltype(stag)::type S;
#define FEW(MP)                                                                                              \
  launch_product4(m.per == 1   ? product4_few_kernel<T, S, MP, 1>                                            \
                  : m.per == 2 ? product4_few_kernel<T, S, MP, 2>                                            \
                               : product4_few_kernel<T, S, MP, 4>,                                           \
                  MP, 16, tx, ty, a, rows, waves, splits, s)
#define MOST2(MT, NT, R)                                                                                     \
  launch_product4(m.per == 1 ? product4_kernel<T, S, MT, NT, R, 1> : product4_kernel<T, S, MT, NT, R, 2>,    \
                  16 * MT, 16 * NT, tx, ty, a, rows, waves, splits, s)
#define MANY(MT, NT, R)                                                                                      \
  launch_product4(m.per == 1   ? product4_kernel<T, S, MT, NT, R, 1>                                         \
                  : m.per == 2 ? product4_kernel<T, S, MT, NT, R, 2>                                         \
                               : product4_kernel<T, S, MT, NT, R, 4>,                                        \
                  16 * MT, 16 * NT, tx, ty, a, rows, waves, splits, s)
      if (src.rows == 1) return FEW(1);
      if (few) return FEW(4);
      // (a shape that is not chosen for four scales has no kernel for them, nor 2 x 4 for two)
      if constexpr (sizeof(T) == 2) {
        if (mt == 3) return MOST2(3, 2, 1);
        if (mt == 2 && nt == 4)
          return launch_product4(product4_kernel<T, S, 2, 4, 1, 1>, 32, 64, tx, ty, a, rows, waves, splits, s);
        if (mt == 2) return nt == 2 ? MANY(2, 2, 1) : MOST2(2, 3, 1);
        return nt == 1 ? MANY(1, 1, 2) : nt == 2 ? MANY(1, 2, 1) : nt == 3 ? MANY(1, 3, 1) : MOST2(1, 4, 2);
      } else {
        if (mt == 2) return MANY(2, 1, 1);
        return nt == 1 ? MANY(1, 1, 1) : MANY(1, 2, 1);
      }
#undef FEW
#undef MANY
#undef MOST2
    });
  });
}

}  // namespace kmhip

using namespace kmhip;

KM_API int h2o4gpu_codebook4_quantize(int dtype, size_t out, size_t cols, int group, float top, const void *d_w,
                                      size_t w_stride, const void *d_codebook, void *d_codes, size_t codes_pitch,
                                      int scale_dtype, void *d_scales, void *stream) {
  if (!known_type(dtype) || out < 1 || out > MOST_ROWS4 || !sizes_ok(1, 1, cols, group) ||
      !packed_ok(d_codes, codes_pitch, cols, scale_dtype, d_scales) || !d_codebook ||
      !aligned_to(d_codebook, type_size(dtype)) || !strided_ok(dtype, d_w, w_stride, cols) || !(top > 0.f) ||
      !isfinite(top))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    return with_type(scale_dtype, [&](auto stag) {
      typedef typename decltype(stag)::type S;
      hipLaunchKernelGGL((quantize4_kernel<T, S>), dim3((unsigned)((out + 3) / 4 < 65536 ? (out + 3) / 4 : 65536)),
                         dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const T *>(d_w),
                         (int64_t)w_stride, (int64_t)out, (int)cols, group, top, static_cast<const T *>(d_codebook),
                         static_cast<uint8_t *>(d_codes), (int64_t)codes_pitch, static_cast<S *>(d_scales));
      return launched();
    });
  });
}

KM_API size_t h2o4gpu_codebook4_codes_bytes(size_t experts, size_t out, size_t cols) {
  return sizes_ok(experts, out, cols, 32) ? experts * tiles_of(out) * subs_of(cols) * 1024 : 0;
}

KM_API size_t h2o4gpu_codebook4_scales_bytes(size_t experts, size_t out, size_t cols, int group, int scale_dtype) {
  if (!sizes_ok(experts, out, cols, group) || !known_type(scale_dtype)) return 0;
  return experts * tiles_of(out) * subs_of(cols) * 16 * scales_per_sub(group) * type_size(scale_dtype);
}

KM_API int h2o4gpu_codebook4_layout(size_t experts, size_t out, size_t cols, int group, const void *d_codes,
                                    size_t codes_pitch, int scale_dtype, const void *d_scales, void *d_laid_codes,
                                    void *d_laid_scales, void *stream) {
  if (!sizes_ok(experts, out, cols, group) || !packed_ok(d_codes, codes_pitch, cols, scale_dtype, d_scales) ||
      !d_laid_codes || !aligned_to(d_laid_codes, 16) || !d_laid_scales || !aligned_to(d_laid_scales, 16))
    return H2O4GPU_KMEANS_EARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t tiles16 = (int64_t)tiles_of(out), lanes = (int64_t)experts * tiles16 * subs_of(cols) * 64;
  hipLaunchKernelGGL(layout4_codes_kernel, dim3(blocks_for(lanes)), dim3(256), 0, s,
                     static_cast<const uint8_t *>(d_codes), (int64_t)codes_pitch, (int64_t)out, (int)cols, tiles16,
                     (int)subs_of(cols), lanes, static_cast<uint4 *>(d_laid_codes));
  KM_TRY(launched());
  const int per = scales_per_sub(group), groups = (int)((cols + group - 1) / group);
  const int64_t count = (int64_t)experts * tiles16 * subs_of(cols) * 16 * per;
  const auto with_scales = [&](auto zero) {
    typedef decltype(zero) S;
    hipLaunchKernelGGL(layout4_scales_kernel<S>, dim3(blocks_for(count)), dim3(256), 0, s,
                       static_cast<const S *>(d_scales), (int64_t)out, groups, group, tiles16, (int)subs_of(cols),
                       per, count, static_cast<S *>(d_laid_scales));
    return launched();
  };
  return scale_dtype == H2O4GPU_EXPERTS_FLOAT32 ? with_scales(0.f) : with_scales((uint16_t)0);
}

// The checks that both products share, and the matrix.
static bool laid_out(int dtype, size_t experts, size_t out, size_t cols, int group, const void *codes,
                     int scale_dtype, const void *scales, const void *book, size_t book_stride, Matrix4 *m) {
  if (!known_type(dtype) || !known_type(scale_dtype) || !sizes_ok(experts, out, cols, group) || !codes ||
      !aligned_to(codes, 16) || !scales || !aligned_to(scales, 16) || !book || !aligned_to(book, type_size(dtype)) ||
      (book_stride != 0 && book_stride < 16) || book_stride > ((size_t)1 << 32))
    return false;
  m->codes = static_cast<const uint4 *>(codes);
  m->scales = scales;
  m->books = book;
  m->book_stride = (int64_t)book_stride;
  m->out = (int64_t)out;
  m->cols = (int)cols;
  m->per = scales_per_sub(group);
  return true;
}

KM_API int h2o4gpu_codebook4_product(int dtype, size_t rows, size_t out, size_t cols, int group, const void *d_x,
                                     size_t x_stride, const void *d_laid_codes, int scale_dtype,
                                     const void *d_laid_scales, const void *d_codebook, void *d_y, size_t y_stride,
                                     void *stream) {
  Matrix4 m;
  if (!laid_out(dtype, 1, out, cols, group, d_laid_codes, scale_dtype, d_laid_scales, d_codebook, 0, &m) ||
      rows > MOST_ROWS4)
    return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!strided_ok(dtype, d_x, x_stride, cols) || !strided_ok(dtype, d_y, y_stride, out)) return H2O4GPU_KMEANS_EARG;
  RowSource src;
  src.rows = (int64_t)rows;
  return product4(dtype, d_x, x_stride, m, scale_dtype, src, d_y, y_stride, static_cast<hipStream_t>(stream));
}

KM_API int h2o4gpu_codebook4_experts_product(int dtype, size_t tokens, int top_k, int experts, size_t out,
                                             size_t cols, int group, const void *d_x, size_t x_stride,
                                             const void *d_laid_codes, int scale_dtype, const void *d_laid_scales,
                                             const void *d_codebook, size_t codebook_stride, const int *d_order,
                                             const int *d_offsets, void *d_y, size_t y_stride, void *stream) {
  Matrix4 m;
  if (experts < 1 ||
      !laid_out(dtype, (size_t)experts, out, cols, group, d_laid_codes, scale_dtype, d_laid_scales, d_codebook,
                codebook_stride, &m) ||
      top_k < 1 || top_k > H2O4GPU_EXPERTS_MAX_TOP_K || tokens > MOST_ROWS4 / (size_t)top_k)
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
  return product4(dtype, d_x, x_stride, m, scale_dtype, src, d_y, y_stride, static_cast<hipStream_t>(stream));
}
