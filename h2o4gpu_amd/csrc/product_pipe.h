// The large tile of a matrix product on gfx950, for operands whose pieces of 16 bytes lie at multiples of 16.
//
// C[m][n] = sum over k of X[m][k] W[n][k], 2-byte and 4-byte elements, or microscaled 4-bit ones (which are handled
// as 2-byte elements that hold four columns each, with their scales beside). A stage of 128 bytes of k for each row
// of both operands goes straight from memory to LDS, into one of two buffers, and is multiplied in two steps. The
// fragments of the next step are read while the matrix instructions of this one run, across the stage's only
// barrier too: at the barrier in the middle of stage t every wavefront holds the rest of stage t in registers, so its
// buffer is free for stage t + 2 from there, and what arrives there is stage t + 1, half a stage before it is needed.
#pragma once

#include <limits.h>

#include "product_tiles.h"

namespace kmhip {

struct Four {};  // as an element type: microscaled 4-bit numbers

enum Kind { FORWARD, DROWS, DWEIGHTS };

struct PipeArgs {
  const char *x, *w;                        // x: m's operand, w: n's
  const unsigned char *x_scales, *w_scales; // Four only, rows of `scales_stride` bytes
  void *c;
  size_t x_stride, w_stride, w_expert, scales_stride;  // bytes
  size_t c_stride, c_expert;                           // elements
  size_t x_bytes;              // GATHER: all of x, below 2^32
  const int *order, *offsets;  // order: x's row of C's row p is order[p] / top_k (none: p)
  int top_k, experts;          // experts 0: one matrix and `rows` rows
  int rows, n, k;              // k in elements (Four: in groups of four columns); DWEIGHTS: k is C's m
  int m_tiles, n_tiles, band;
  int c_aligned;               // C's rows begin at multiples of 16 bytes
};

template <typename T>
struct PipeElement {
  typedef T type;
};
template <>
struct PipeElement<Four> {
  typedef bfloat16_t type;
};

template <typename T>
struct Pieces {
  T v[16 / sizeof(T)];
};

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ unsigned lds_address(const void *p) {
  return (unsigned)(size_t)(lds_char *)(const_cast<void *>(p));
}
__device__ __forceinline__ u32x4 lds_read_16(unsigned at) {
  return *(__attribute__((address_space(3))) const u32x4 *)(size_t)at;
}
__device__ __forceinline__ unsigned lds_read_4(unsigned at) {
  return *(__attribute__((address_space(3))) const unsigned *)(size_t)at;
}
__device__ __forceinline__ u32x2 lds_read_turned(unsigned at) {
  u32x2 out = {at, at};
#if defined(__HIP_DEVICE_COMPILE__)
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  out = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(size_t)at));
#endif
  return out;
}
// A pointer that is the same in every lane, for the compiler to see.
__device__ __forceinline__ const char *same_in_all(const char *p) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)(size_t)p);
  const unsigned hi = __builtin_amdgcn_readfirstlane((unsigned)((size_t)p >> 32));
  return (const char *)((size_t)hi << 32 | lo);
}
// 16 bytes at each lane's own offset behind a buffer's start to 64 consecutive places from `lds` on (the same in every
// lane); nothing is read behind the buffer's size. Written out, because the compiler would wait for all of these before
// a read of LDS that it cannot tell from where they write; who reads there waits for vmcnt by hand.
__device__ __forceinline__ u32x4 buffer_of(const char *start, unsigned size) {
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(size_t)start),
               (unsigned)__builtin_amdgcn_readfirstlane((unsigned)((size_t)start >> 32) & 0xffffu),
               (unsigned)__builtin_amdgcn_readfirstlane(size), 0x00020000u};
}
__device__ __forceinline__ void to_lds_16(u32x4 buffer, unsigned offset, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(offset), "s"(buffer));
#endif
}

// The scales' bytes are number SELECT of their words. Written out, because only so the sum stays in its registers (the
// compiler gives the builtin's result others, and spills where all are taken). It knows no waits for it: a sum is
// touched by nothing but these until sums_done(), and again by one only 15 others later.
template <int SELECT>
__device__ __forceinline__ void mfma_four(f32x4 &acc, u32x4 w, u32x4 x, unsigned sw, unsigned sx) {
#if defined(__HIP_DEVICE_COMPILE__)
#define KM_MFMA_FOUR(MORE)                                                                               \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " MORE " cbsz:4 blgp:4" \
               : "+v"(acc)                                                                               \
               : "v"(w), "v"(x), "v"(sw), "v"(sx))
  if constexpr (SELECT == 0) KM_MFMA_FOUR("op_sel_hi:[0,0,0]");
  if constexpr (SELECT == 1) KM_MFMA_FOUR("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  if constexpr (SELECT == 2) KM_MFMA_FOUR("op_sel_hi:[1,1,0]");
  if constexpr (SELECT == 3) KM_MFMA_FOUR("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef KM_MFMA_FOUR
#endif
}
// The matrix instructions before it have written their sums.
template <int FM, int FN>
__device__ __forceinline__ void sums_done(f32x4 (&acc)[FM][FN]) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) asm volatile("" : "+v"(acc[i][j]));
#endif
}

// One operand of a tile of R rows in a workgroup of THREADS: where its pieces come from, where fragments lie.
template <typename T, int R, bool COLUMNS, int THREADS, int F>
struct PipeOperand {
  typedef OperandTile<T, R, COLUMNS> Tile;
  static constexpr int P = Tile::SLOTS / THREADS, SIZE = (int)sizeof(T);
  static constexpr int ADDRESSES = !COLUMNS ? 2 : sizeof(T) == 2 ? F : 1;
  static constexpr int READS = !COLUMNS ? 1 : sizeof(T) == 2 ? 2 : 4;  // LDS reads of a fragment
  unsigned at[ADDRESSES];  // of this wavefront's fragments, in the buffer that is read

  __device__ __forceinline__ void init(unsigned lds, int lane, int block0) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!COLUMNS) {
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = lds + ((block0 * 16 + i) * 8 + ((s * 4 + g) ^ (i & 7))) * 16;
    } else if constexpr (sizeof(T) == 2) {
      const int k = 8 * g + (i >> 2);
#pragma unroll
      for (int b = 0; b < F; ++b)
        at[b] = lds + (k * Tile::PER_K + ((2 * (block0 + b) + ((i & 3) >> 1)) ^ Tile::turn(k))) * 16 + (i & 1) * 8;
    } else {
      at[0] = lds + 4 * g * Tile::PER_K * 16 + ((4 * block0 + (i >> 2)) ^ (4 * g)) * 16 + (i & 3) * 4;
    }
  }
  __device__ __forceinline__ void swap(unsigned bit) {
#pragma unroll
    for (int i = 0; i < ADDRESSES; ++i) at[i] ^= bit;
  }
  template <int STEP>
  __device__ __forceinline__ u32x4 fragment(int b) const {
    if constexpr (!COLUMNS) {
      return lds_read_16(at[STEP] + b * 2048);
    } else if constexpr (sizeof(T) == 2) {
      constexpr int LINE = Tile::PER_K * 16;
      const u32x2 lo = lds_read_turned(at[b] + STEP * 32 * LINE), hi = lds_read_turned(at[b] + (STEP * 32 + 4) * LINE);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      // (turn(k) is 4 g for k = 16 step + 4 g + j, and 4 b flips the same bits of the piece)
      constexpr int LINE = Tile::PER_K * 16;
      u32x4 out;
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = lds_read_4((at[0] ^ (b * 64)) + (STEP * 16 + j) * LINE);
      return out;
    }
  }
};

constexpr int PIPE_TABLE = 2046;  // experts + 2 numbers of 4 bytes fit 8 KB of LDS

// table[e]: how many tiles of BM rows the experts before e have; [experts + 1]: all, those without an expert included.
template <int BM, int THREADS>
__device__ __forceinline__ void tile_table(int *table, const int *offsets, int experts, int rows) {
  constexpr int EACH = (PIPE_TABLE + 1 + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int mine[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = tid * EACH + i;
    mine[i] = 0;
    if (e <= experts) mine[i] = ((e < experts ? offsets[e + 1] : rows) - offsets[e] + BM - 1) / BM;
    sum += mine[i];
  }
  int before = sum;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int other = __shfl_up(before, d);
    if (lane >= d) before += other;
  }
  // (the sums of whole wavefronts lie behind the table)
  int *sums = table + PIPE_TABLE + 2;
  if (lane == 63) sums[wave] = before;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < wave; ++w) before += sums[w];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = tid * EACH + i;
    if (e <= experts) table[e] = before;
    before += mine[i];
    if (e == experts) table[e + 1] = before;
  }
  __syncthreads();
}

template <int BM>
__device__ __forceinline__ void listed_tile(const int *table, const int *offsets, int experts, int rows, int number,
                                            int &stretch, int &first, int &rows_here) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = experts + 1;  // the last e with table[e] <= number
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool below = lane * step < n && table[lo + lane * step] <= number;
    const int skip = (__popcll(__ballot(below)) - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int begin = offsets[lo], end = lo == experts ? rows : offsets[lo + 1];
  stretch = lo;
  first = begin + (number - __builtin_amdgcn_readfirstlane(table[lo])) * BM;
  rows_here = end - first < BM ? end - first : BM;
}

// A wavefront's part of a tile to memory: through its own LDS, so that a row's numbers go out side by side, 16 bytes a
// lane. (The lanes of a sum hold four numbers of 16 rows each; stored as they are, 8192^3 took 100 us longer.)
template <typename OUT, int FM, int FN, int BYTES>
__device__ __forceinline__ void store_tile(char *mine, int lane, f32x4 (&acc)[FM][FN], OUT *c, size_t stride, int m0,
                                           int n0, int m_here, int n_here, bool aligned) {
  constexpr int LINE = FN * 16 * (int)sizeof(OUT), PIECES = LINE / 16, EPP = 16 / (int)sizeof(OUT);
  constexpr int PASS = BYTES / (LINE * 16) < FM ? BYTES / (LINE * 16) : FM;  // blocks of 16 rows at a time
  static_assert(PASS >= 1 && FM % PASS == 0 && PIECES >= 8 && 64 % PIECES == 0, "");
  if (!aligned) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + i * 16 + (lane & 15);
      if (m >= m_here) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = n0 + j * 16 + 4 * (lane >> 4);
        store_four(c + (size_t)m * stride + n, acc[i][j], n_here - n, false);
      }
    }
    return;
  }
#pragma unroll
  for (int p = 0; p < FM / PASS; ++p) {
#pragma unroll
    for (int i = 0; i < PASS; ++i) {
      const int m = i * 16 + (lane & 15);
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int byte = (j * 16 + 4 * (lane >> 4)) * (int)sizeof(OUT);
        char *at = mine + m * LINE + (byte / 16 ^ (m & 7)) * 16 + byte % 16;
        store_four(reinterpret_cast<OUT *>(at), acc[p * PASS + i][j], 4, true);
      }
    }
#pragma unroll
    for (int r = 0; r < PASS * 16 * PIECES / 64; ++r) {
      const int m = r * (64 / PIECES) + lane / PIECES, piece = lane % PIECES;
      const u32x4 v = *reinterpret_cast<const u32x4 *>(mine + m * LINE + (piece ^ (m & 7)) * 16);
      const int row = m0 + p * PASS * 16 + m, n = n0 + piece * EPP;
      if (row < m_here && n < n_here) {
        OUT *to = c + (size_t)row * stride + n;
        if (n + EPP <= n_here) {
          *reinterpret_cast<u32x4 *>(to) = v;
        } else {
#pragma unroll
          for (int e = 0; e < EPP; ++e)
            if (n + e < n_here) to[e] = __builtin_bit_cast(Pieces<OUT>, v).v[e];
        }
      }
    }
  }
}

template <typename ELEMENT, typename OUT, Kind KIND, bool GATHER, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64) void pipe_kernel(PipeArgs a) {
  typedef typename PipeElement<ELEMENT>::type T;
  constexpr bool FOUR = __is_same(ELEMENT, Four);
  constexpr bool XC = KIND == DWEIGHTS, WC = KIND != FORWARD;
  constexpr int THREADS = WM * WN * 64;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  typedef PipeOperand<T, BM, XC, THREADS, FM> X;
  typedef PipeOperand<T, BN, WC, THREADS, FN> W;
  constexpr int SIZE = (int)sizeof(T), EPP = 16 / SIZE, KS = 8 * EPP;
  constexpr int STAGE = (BM + BN) * 128;
  static_assert((STAGE & (STAGE - 1)) == 0, "the buffers are told apart by one bit");
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Tiles of m, numbered without gaps: those of expert 0, of expert 1, ..., of the rows without an expert. A table in
  // LDS says where each expert's begin; beyond PIPE_TABLE experts the numbers have gaps (ragged_tile).
  int *table = reinterpret_cast<int *>(lds + 2 * STAGE + (FOUR ? 2 * (BM + BN) * 16 : 0));
  const bool ragged = KIND != DWEIGHTS && a.experts > 0, listed = ragged && a.experts < PIPE_TABLE;
  unsigned m_tiles = (unsigned)a.m_tiles;
  if (listed) {
    tile_table<BM, THREADS>(table, a.offsets, a.experts, a.rows);
    m_tiles = __builtin_amdgcn_readfirstlane(table[a.experts + 1]);
  }
  // Workgroups go round the eight chiplets; each of these takes a stretch of the tiles, and its workgroups neighbours
  // of that at the same time: `band` tiles of m by as many of n as there are workgroups.
  const unsigned total = m_tiles * (unsigned)a.n_tiles, die = blockIdx.x & 7;
  const unsigned last_tile = (unsigned)((unsigned long long)total * (die + 1) / 8);
  for (unsigned tile = (unsigned)((unsigned long long)total * die / 8) + (blockIdx.x >> 3); tile < last_tile;
       tile += gridDim.x >> 3) {
  // (what follows from a thread's number is made anew for each tile and each part of it: kept, it would take the
  // registers of the sums)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  int number, n_tile;
  {
    const unsigned band = (unsigned)a.band * a.n_tiles, m0 = tile / band * a.band;
    const unsigned high = m_tiles - m0 < (unsigned)a.band ? m_tiles - m0 : a.band;
    const unsigned in = tile % band;
    number = (int)(m0 + in % high), n_tile = (int)(in / high);
  }
  const int n0 = n_tile * BN, n_here = a.n - n0 < BN ? a.n - n0 : BN;
  int expert = 0, first = number * BM, m_here, k_end = a.k;
  const char *x = a.x, *w = a.w;
  OUT *c = static_cast<OUT *>(a.c);
  if constexpr (KIND == DWEIGHTS) {
    const int tiles = (a.k + BM - 1) / BM;
    expert = number / tiles, first = number % tiles * BM;
    m_here = a.k - first < BM ? a.k - first : BM;
    const int begin = a.offsets[expert];
    k_end = a.offsets[expert + 1] - begin;
    x += (size_t)begin * a.x_stride + (size_t)first * SIZE;
    w += (size_t)begin * a.w_stride + (size_t)n0 * SIZE;
    c += (size_t)expert * a.c_expert + (size_t)first * a.c_stride;
  } else {
    m_here = a.rows - first < BM ? a.rows - first : BM;
    if (ragged) {
      if (listed)
        listed_tile<BM>(table, a.offsets, a.experts, a.rows, number, expert, first, m_here);
      else if (!ragged_tile(a.offsets, a.experts, a.rows, BM, number, expert, first, m_here))
        continue;
      if (expert == a.experts) k_end = 0, expert = 0;  // rows without an expert: zeros
    }
    if (!GATHER) x += (size_t)first * a.x_stride;
    w += (size_t)expert * a.w_expert + (WC ? (size_t)n0 * SIZE : (size_t)n0 * a.w_stride);
    c += (size_t)first * a.c_stride;
  }
  const int stages = (k_end + KS - 1) / KS, full = k_end / KS;

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wm = wave / WN, wn = wave % WN;

  if (stages > 0) {
    // Where a lane's pieces lie behind a stage's start. No piece is clamped: what lies behind the operand's last byte
    // of the stage is not read, and a piece of a row or column that does not exist is multiplied into what is not
    // stored, or masked.
    unsigned x_off[GATHER ? X::P : 1], w_off;
    {
      int r, k;
      W::Tile::place(tid, r, k);
      w_off = WC ? (unsigned)(k * a.w_stride) + r * SIZE : (unsigned)(r * a.w_stride) + k * SIZE;
#pragma unroll
      for (int i = 0; i < (GATHER ? X::P : 1); ++i) {
        X::Tile::place(i * THREADS + tid, r, k);
        if (GATHER) {
          const int p = first + (r < m_here ? r : m_here - 1);
          x_off[i] = (unsigned)((a.order[p] / a.top_k) * a.x_stride) + k * SIZE;
        } else {
          x_off[i] = XC ? (unsigned)(k * a.x_stride) + r * SIZE : (unsigned)(r * a.x_stride) + k * SIZE;
        }
      }
    }
    // from one of a lane's pieces to its next: THREADS slots on are so many rows or k on, turned alike
    const unsigned x_next = (unsigned)((XC ? THREADS / X::Tile::PER_K : THREADS / 8) * a.x_stride);
    const unsigned w_next = (unsigned)((WC ? THREADS / W::Tile::PER_K : THREADS / 8) * a.w_stride);
    const size_t x_step = XC ? KS * a.x_stride : 128, w_step = WC ? KS * a.w_stride : 128;
    // Scales of two stages (512 columns), 16 bytes a row: the first BM lanes of the workgroup load x's, BN others w's.
    constexpr int SCALES = (BM + BN) * 16;
    static_assert(!FOUR || BM + BN == THREADS || BM + BN == 2 * THREADS, "a lane loads one or two rows' scales");
    constexpr int PS = FOUR ? (BM + BN) / THREADS : 1;
    unsigned s_off[PS], s_size[PS];
    const char *s_from[PS];
    if constexpr (FOUR) {
#pragma unroll
      for (int i = 0; i < PS; ++i) {
        const bool of_x = i * THREADS + wave * 64 < BM;
        const size_t row = of_x ? (GATHER ? 0 : (size_t)first) : (size_t)expert * a.n + n0;
        const unsigned rows = of_x ? (GATHER ? (unsigned)(a.x_bytes / a.x_stride) : (unsigned)m_here) : (unsigned)n_here;
        s_from[i] = same_in_all((const char *)(of_x ? a.x_scales : a.w_scales) + row * a.scales_stride);
        s_size[i] = __builtin_amdgcn_readfirstlane((rows - 1) * (unsigned)a.scales_stride + 16);
        const int r = i * THREADS + tid;
        if (GATHER && r < BM) {
          const int m = r < m_here ? r : m_here - 1;
          s_off[i] = (unsigned)((a.order[first + m] / a.top_k) * a.scales_stride);
        } else {
          s_off[i] = (unsigned)((r < BM ? r : r - BM) * a.scales_stride);
        }
      }
    }
    const unsigned base = lds_address(lds), to = base + wave * 1024;
    auto load_scales = [&](int pair) {
      if constexpr (FOUR) {
        const unsigned s = to + 2 * STAGE + (pair & 1) * SCALES;
#pragma unroll
        for (int i = 0; i < PS; ++i) {
          to_lds_16(buffer_of(s_from[i] + (size_t)pair * 16, pair * 2 < stages ? s_size[i] : 0), s_off[i], s + i * THREADS * 16);
        }
      }
    };
    // The stage that is loaded next, and how much of it there is.
    struct Stage {
      const char *x, *w;
      unsigned x_size, w_size, to;
    } next;
    const auto x_size_of = [&](int k_here) {
      return XC ? (unsigned)((k_here - 1) * a.x_stride) + m_here * SIZE : (unsigned)((m_here - 1) * a.x_stride) + k_here * SIZE;
    };
    const auto w_size_of = [&](int k_here) {
      return WC ? (unsigned)((k_here - 1) * a.w_stride) + n_here * SIZE : (unsigned)((n_here - 1) * a.w_stride) + k_here * SIZE;
    };
    const unsigned x_full = x_size_of(KS), w_full = w_size_of(KS);
    const unsigned x_last = x_size_of(k_end - full * KS), w_last = w_size_of(k_end - full * KS);
    unsigned x_left = GATHER ? (unsigned)a.x_bytes : 0;
    auto size_next = [&](int t) {
      next.x_size = t < full ? (GATHER ? x_left : x_full) : t < stages ? x_last : 0;
      next.w_size = t < full ? w_full : t < stages ? w_last : 0;
    };
    next.x = x, next.w = w, next.to = to;
    size_next(0);
    auto advance = [&](int t) {  // to stage t
      next.x += x_step, next.w += w_step, next.to ^= STAGE;
      if (GATHER) x_left -= 128;
      size_next(t);
    };
    auto load_one = [&](int i) {
      if (i < X::P)
        to_lds_16(buffer_of(next.x, next.x_size), GATHER ? x_off[GATHER ? i : 0] : x_off[0] + i * x_next,
                  next.to + i * THREADS * 16);
      else
        to_lds_16(buffer_of(next.w, next.w_size), w_off + (i - X::P) * w_next,
                  next.to + BM * 128 + (i - X::P) * THREADS * 16);
    };
    auto load = [&]() {
#pragma unroll
      for (int i = 0; i < X::P + W::P; ++i) load_one(i);
    };
    X fx;
    W fw;
    fx.init(base, lane, wm * FM);
    fw.init(base + BM * 128, lane, wn * FN);
    const unsigned s_at = base + 2 * STAGE + (lane & 15) * 16 + 4 * (lane >> 4);

    struct Fragments {
      u32x4 x[FM], w[FN];
    } f[2];
    auto read_one = [&](auto step, int r) {
      constexpr int S = decltype(step)::value;
      if (r < FN)
        f[S].w[r] = fw.template fragment<S>(r);
      else
        f[S].x[r - FN] = fx.template fragment<S>(r - FN);
    };
    auto read = [&](auto step) {
#pragma unroll
      for (int r = 0; r < FN + FM; ++r) read_one(step, r);
    };
    unsigned sx[FOUR ? FM : 1], sw[FOUR ? FN : 1];
    auto read_scales = [&](int pair) {
      if constexpr (FOUR) {
        const unsigned s = s_at + (pair & 1) * SCALES;
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] = lds_read_4(s + (wm * FM + i) * 256);
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] = lds_read_4(s + BM * 16 + (wn * FN + j) * 256);
      }
    };
    // product q of a step of a stage of even (ODD 0) or odd number
    auto multiply_one = [&](auto step, auto odd, int q) {
      constexpr int S = decltype(step)::value, ODD = decltype(odd)::value;
      const int i = q / FN, j = q % FN;
      if constexpr (FOUR)
        mfma_four<2 * ODD + S>(acc[i][j], f[S].w[j], f[S].x[i], sw[j], sx[i]);
      else
        mfma_piece(acc[i][j], f[S].w[j], f[S].x[i], Tag<T>());
    };
    // A step's products, with `reads` LDS reads spread between the first 3/4 of them and `loads` loads between all. (A
    // load takes its turn in the CU's address unit; a wavefront that has to wait for that issues nothing else.)
    auto multiply = [&](auto step, auto odd, auto reads, auto read_it, auto loads, auto load_it) {
      constexpr int R = decltype(reads)::value, L = decltype(loads)::value, Q = FM * FN, SPAN = Q * 3 / 4;
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        // (the r-th goes before product r * SPAN / R)
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (r * SPAN / (R ? R : 1) == q) read_it(r);
#pragma unroll
        for (int l = 0; l < L; ++l)
          if (l * Q / (L ? L : 1) == q) load_it(l);
        multiply_one(step, odd, q);
        if (R || L) __builtin_amdgcn_sched_barrier(0);
      }
    };
    // everything this wavefront has asked for is there; then everybody's is
    auto meet = [&]() {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    // A step that reaches behind the last k: what lies there is no part of the sum, and may be anything.
    auto mask = [&](auto step) {
      constexpr int S = decltype(step)::value;
      const int left = k_end - full * KS - S * (KS / 2) - EPP * (lane >> 4);
      if (left < EPP) {
        u32x4 keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int bytes = (left * SIZE) - 4 * i;
          keep[i] = bytes >= 4 ? 0xffffffffu : bytes <= 0 ? 0u : 0xffffu;
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) f[S].x[i] &= keep;
#pragma unroll
        for (int j = 0; j < FN; ++j) f[S].w[j] &= keep;
      }
    };

    load();
    load_scales(0);
    meet();
    advance(1);
    load();
    read(Int<0>());
    read_scales(0);
    constexpr int LOADS = X::P + W::P, READS = FM + FN;
    auto stage = [&](int t, auto odd) {
      multiply(Int<0>(), odd, Int<READS>(), [&](int r) { read_one(Int<1>(), r); }, Int<0>(), [](int) {});
      advance(t + 2);
      meet();
      if (!decltype(odd)::value) load_scales((t >> 1) + 1);
      fx.swap(STAGE), fw.swap(STAGE);
      multiply(
          Int<1>(), odd, Int<READS>(), [&](int r) { read_one(Int<0>(), r); }, Int<LOADS>(),
          [&](int l) { load_one(l); });
      if (decltype(odd)::value) read_scales((t >> 1) + 1);
    };
    if constexpr (FOUR) {
      for (int t = 0;;) {
        stage(t, Int<0>());
        if (++t == stages) break;
        stage(t, Int<1>());
        if (++t == stages) break;
      }
      sums_done(acc);
    } else {
      for (int t = 0; t < full; ++t) stage(t, Int<0>());
    }
    if (!FOUR && full < stages) {
      read(Int<1>());
      mask(Int<0>());
      multiply(Int<0>(), Int<0>(), Int<0>(), [](int) {}, Int<0>(), [](int) {});
      mask(Int<1>());
      multiply(Int<1>(), Int<0>(), Int<0>(), [](int) {}, Int<0>(), [](int) {});
    }
  }
  // loads that read nothing end, and everybody's reads, before the LDS is used again
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();

  int tid2 = threadIdx.x;
  asm volatile("" : "+v"(tid2));
  store_tile<OUT, FM, FN, STAGE * 2 / (WM * WN)>(lds + wave * (STAGE * 2 / (WM * WN)), tid2 & 63, acc, c + n0, a.c_stride,
                                                 wm * FM * 16, wn * FN * 16, m_here, n_here, a.c_aligned);
  __syncthreads();
  }
}

constexpr size_t PIPE_WORKGROUPS = 256;    // one to a CU, as many as the LDS allows
constexpr size_t BUFFER_BYTES = (size_t)1 << 32;  // what a buffer's offsets reach

template <typename ELEMENT, typename OUT, Kind KIND, bool GATHER, int BM, int BN, int WM, int WN>
int launch_pipe(PipeArgs &a, hipStream_t stream) {
  const size_t m_tiles = KIND == DWEIGHTS ? (size_t)a.experts * ((a.k + BM - 1) / BM)
                         : a.experts      ? ragged_tiles(a.experts, a.rows, BM)
                                          : ((size_t)a.rows + BM - 1) / BM;
  a.m_tiles = (int)m_tiles, a.n_tiles = (a.n + BN - 1) / BN;
  a.band = a.n_tiles >= 8 ? 4 : a.n_tiles >= 4 ? 8 : 16;
  const size_t tiles = m_tiles * a.n_tiles;
  if (m_tiles > (size_t)INT_MAX || tiles > (size_t)INT_MAX) return H2O4GPU_KMEANS_EARG;
  const size_t lds = (BM + BN) * (256 + (__is_same(ELEMENT, Four) ? 32 : 0)) + (PIPE_TABLE + 2 + WM * WN) * 4;
  const auto kernel = pipe_kernel<ELEMENT, OUT, KIND, GATHER, BM, BN, WM, WN>;
  KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds));
  const size_t blocks = tiles < PIPE_WORKGROUPS ? (tiles + 7) / 8 * 8 : PIPE_WORKGROUPS;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(WM * WN * 64), lds, stream, a);
  return launched();
}

}  // namespace kmhip
