// The large tiles of a matrix product on gfx950, for operands whose rows begin at multiples of 4 bytes.
//
// C[m][n] = sum over k of X[m][k] W[n][k], 2-byte and 4-byte elements, or microscaled 4-bit ones (which are handled
// as 2-byte elements that hold four columns each, with their scales beside). A stage of 128 bytes of k for each row
// of both operands goes straight from memory to LDS, into one of two buffers, and is multiplied in two steps. The
// fragments of the next step are read while the matrix instructions of this one run, across the stage's only
// barrier too: at the barrier in the middle of stage t every wavefront holds the rest of stage t in registers, so its
// buffer is free for stage t + 2 from there, and what arrives there is stage t + 1, half a stage before it is needed.
#pragma once

#include "product_tiles.h"

namespace kmhip {

struct Four {};  // as an element type: microscaled 4-bit numbers

struct PipeArgs {
  const char *x, *w;                        // x: m's operand, w: n's
  const unsigned char *x_scales, *w_scales; // Four only, rows of `scales_stride` bytes
  void *c;
  size_t x_stride, w_stride, w_expert, scales_stride;  // bytes
  size_t c_stride, c_expert;                           // elements
  size_t x_bytes;              // GATHER: all of x, below 2^32
  const int *order, *offsets;  // order: x's row of C's row p is order[p] / top_k (none: p)
  int part;                    // DWEIGHTS: rows of a part of an expert's (PartOfRows)
  float *sums;
  int top_k, experts;          // experts 0: one matrix and `rows` rows
  int rows, n, k;              // k in elements (Four: in groups of four columns); DWEIGHTS: k is C's m
  int m_tiles, n_tiles, band;
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
// the other one of two places `apart` bytes apart, the first at `start`
__device__ __forceinline__ unsigned scales_swapped(unsigned at, unsigned apart, unsigned start) {
  return at >= start + apart ? at - apart : at + apart;
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
// a read of LDS that it cannot tell from where they write; who reads there waits for vmcnt by hand. That is also why no
// memory is named as changed: stages and scales are read behind meet(), which is a barrier to the compiler too, and which
// every load has behind it before its stage is read; before the first stages it is s_waitcnt and __syncthreads(). (Row
// numbers are ordinary stores.) The compiler does not look in here either for the five states that a memory instruction has
// to stay behind a vector instruction, as readfirstlane is, that wrote one of its scalar registers: settled() is called
// where a buffer's start or size may come from such, once for a tile. (Waiting here, for every load, cost 800 x 2048 x 8192
// in 4 bits 57 -> 60 us.) m0 is named, so that no value of the compiler's own is kept there; it warns of every such name,
// since it gives m0 to no variable.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ u32x4 buffer_of(const char *start, unsigned size) {
  return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(size_t)start),
               (unsigned)__builtin_amdgcn_readfirstlane((unsigned)((size_t)start >> 32) & 0xffffu),
               (unsigned)__builtin_amdgcn_readfirstlane(size), 0x00020000u};
}
__device__ __forceinline__ void to_lds_16(u32x4 buffer, unsigned offset, unsigned lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(offset), "s"(buffer)
               : "m0");
#endif
}
#pragma clang diagnostic pop
// A memory instruction may read these scalar registers, whatever wrote them.
__device__ __forceinline__ void settled(const char *&a, const char *&b) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 4" : "+s"(a), "+s"(b));
#endif
}
__device__ __forceinline__ void settled(const char *&start, unsigned &size) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_nop 4" : "+s"(start), "+s"(size));
#endif
}

// The scales' bytes are number SELECT of their words.
template <int SELECT>
__device__ __forceinline__ void mfma_four(f32x4 &acc, u32x4 w, u32x4 x, unsigned sw, unsigned sx) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef int i32x8 __attribute__((ext_vector_type(8)));
  const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  const i32x8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, SELECT, (int)sw, SELECT, (int)sx);
  asm volatile("" : "+v"(acc));  // (stays where it is written, between the loads around it)
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

constexpr int PIPE_TABLE = 1022;  // experts + 2 numbers of 4 bytes fit 4 KB of LDS

// table[e]: the sum of count(rows of an expert) over the experts before e; [experts + 1]: over all, and over the rows
// without an expert.
template <int THREADS, typename COUNT>
__device__ __forceinline__ void tile_table(int *table, const int *offsets, int experts, int rows, COUNT count) {
  constexpr int EACH = (PIPE_TABLE + 1 + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int mine[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = tid * EACH + i;
    mine[i] = 0;
    if (e <= experts) mine[i] = count((e < experts ? offsets[e + 1] : rows) - offsets[e]);
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

// The last e of the first `n` with table[e] <= number.
__device__ __forceinline__ int last_below(const int *table, int n, int number) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const bool below = lane * step < n && table[lo + lane * step] <= number;
    const int skip = (__popcll(__ballot(below)) - 1) * step;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

template <int BM>
__device__ __forceinline__ void listed_tile(const int *table, const int *offsets, int experts, int rows, int number,
                                            int &stretch, int &first, int &rows_here) {
  const int lo = last_below(table, experts + 1, number);
  const int begin = offsets[lo], end = lo == experts ? rows : offsets[lo + 1];
  stretch = lo;
  first = begin + (number - __builtin_amdgcn_readfirstlane(table[lo])) * BM;
  rows_here = end - first < BM ? end - first : BM;
}

// A wavefront's part of a tile to memory, 16 bytes a lane and 64 of a row side by side. A lane has four numbers of a row;
// of 2-byte ones, the quarters of the wavefront (16 lanes) that hold neighbours exchange halves of two blocks: what bit 0
// of the block's number and the two of the quarter's say (b; q1 q0) lies after the first exchange at (q1; b q0), after
// the second at (q0; b q1). (Stored as they are, eight bytes a lane, 8192^3 in 4 bits takes 265 us instead of 245, and
// 64 experts' 64000 rows of 512 with 512 x 512, bfloat16, 45 instead of 37.)
template <typename OUT, int FM, int FN>
__device__ __forceinline__ void store_tile(int lane, const f32x4 (&acc)[FM][FN], OUT *c, size_t stride, int m0, int n0,
                                           int m_here, int n_here) {
  constexpr int EPP = 16 / (int)sizeof(OUT);
  const int i = lane & 15, q = lane >> 4;
#pragma unroll
  for (int b = 0; b < FM; ++b) {
    const int m = m0 + b * 16 + i;
    OUT *row = c + (size_t)m * stride;
    if constexpr (sizeof(OUT) == 4) {
      if (m < m_here) {
#pragma unroll
        for (int j = 0; j < FN; ++j) store_four(row + n0 + j * 16 + 4 * q, acc[b][j], n_here - (n0 + j * 16 + 4 * q));
      }
    } else {
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        typedef OUT four __attribute__((ext_vector_type(4)));
        u32x2 lo = __builtin_bit_cast(u32x2, four{(OUT)acc[b][j][0], (OUT)acc[b][j][1], (OUT)acc[b][j][2], (OUT)acc[b][j][3]});
        u32x2 hi = __builtin_bit_cast(
            u32x2, four{(OUT)acc[b][j + 1][0], (OUT)acc[b][j + 1][1], (OUT)acc[b][j + 1][2], (OUT)acc[b][j + 1][3]});
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const auto far = __builtin_amdgcn_permlane32_swap(lo[w], hi[w], false, false);
          const auto near = __builtin_amdgcn_permlane16_swap(far[0], far[1], false, false);
          lo[w] = near[0], hi[w] = near[1];
        }
#endif
        const u32x4 piece = {lo[0], lo[1], hi[0], hi[1]};
        const int n = n0 + j * 16 + 8 * q;
        if (m < m_here && n < n_here) {
          if (n + EPP <= n_here) {
            store_beside<OUT, EPP>(row + n, __builtin_bit_cast(typename Beside<OUT, EPP>::vector, piece));
          } else {
#pragma unroll
            for (int e = 0; e < EPP; ++e)
              if (n + e < n_here) row[n + e] = __builtin_bit_cast(Pieces<OUT>, piece).v[e];
          }
        }
      }
    }
  }
}

// One stage after another, of one tile after another: what is loaded is two stages ahead of what is multiplied, and may be
// the next tile's, so that a tile's first stages arrive while the one before ends and goes out.
//
// Bound by the matrix instructions, and for random numbers by the clock that the card's power leaves: 8192^3 in bfloat16
// takes 790 to 910 us (1200 to 1390 TFLOP/s; zeros 740), in 4 bits 245 (4500; zeros 201), 8192 x 4096 x 4096 in float32
// 1850 (149). 64 experts' 65536 rows of 2048 with 2048 x 2048 take 493 us, the rows' gradient 491, the matrices' 531
// (1115, 1120 and 1035 TFLOP/s). With few columns a tile's way out counts: 64 experts' 65536 rows of 2048 with 4096 x 2048
// in 4 bits take 402 us, of which 105 are for y's 537 MB. A tile of 256 x 256 reads each of its operands' elements from
// LDS as often as there are wavefronts beside it, twice and four times: what eight wavefronts read in a step takes three
// quarters of the time of their matrix instructions. Four of 128 x 128 would read two thirds of that, but the sums leave
// them too few registers.
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
  constexpr int STAGE = (BM + BN) * 128, SCALES = (BM + BN) * 16;
  static_assert((STAGE & (STAGE - 1)) == 0, "the buffers are told apart by one bit");
  static_assert(!FOUR || BM + BN == THREADS, "a lane loads one row's scales");
  // stages, two of them | Four: scales of two stages, two of these | GATHER: which rows of x, of two tiles | table of tiles
  extern __shared__ __attribute__((aligned(16))) char lds[];
  unsigned *gathered = reinterpret_cast<unsigned *>(lds + 2 * STAGE + (FOUR ? 2 * SCALES : 0));
  int *table = reinterpret_cast<int *>(gathered + (GATHER ? 2 * BM : 0));

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const unsigned base = lds_address(lds), to = base + wave * 1024;
  // Tiles of m are numbered without gaps: those of expert 0, of expert 1, ..., of the rows without an expert. A table in
  // LDS says where each expert's begin; beyond PIPE_TABLE experts the numbers have gaps (ragged_tile).
  const bool in_parts = KIND == DWEIGHTS && a.part < a.rows;
  const bool ragged = KIND != DWEIGHTS && a.experts > 0, listed = a.experts > 0 && a.experts < PIPE_TABLE && !in_parts;
  auto stages_of = [](int k) { return k <= KS ? 2 : (k + KS - 1) / KS; };
  unsigned m_tiles = (unsigned)a.m_tiles;
  // Workgroups go round the eight chiplets; each of these takes a stretch of the tiles, and its workgroups neighbours
  // of that at the same time: `band` tiles of m by as many of n as there are workgroups.
  const unsigned die = blockIdx.x & 7;
  unsigned tile, tiles_end;
  if (listed && KIND == DWEIGHTS) {
    // stretches of as many stages, since an expert's tiles have as many as its rows fill
    tile_table<THREADS>(table, a.offsets, a.experts, a.rows, stages_of);
    const unsigned long long each = m_tiles / a.experts * (unsigned)a.n_tiles, all = table[a.experts] * each;
    auto border = [&](unsigned d) {
      const unsigned long long work = all * d / 8;
      const int e = last_below(table, a.experts, (int)(work / each));
      const unsigned stages = table[e + 1] - table[e];
      const unsigned long long in = (work - table[e] * each) / stages;
      return (unsigned)__builtin_amdgcn_readfirstlane((int)(e * each + (in < each ? in : each)));
    };
    tile = border(die) + (blockIdx.x >> 3), tiles_end = border(die + 1);
  } else {
    if (listed) {
      tile_table<THREADS>(table, a.offsets, a.experts, a.rows, [](int rows) { return (rows + BM - 1) / BM; });
      m_tiles = __builtin_amdgcn_readfirstlane(table[a.experts + 1]);
    }
    const unsigned total = m_tiles * (unsigned)a.n_tiles;
    tiles_end = (unsigned)((unsigned long long)total * (die + 1) / 8);
    tile = (unsigned)((unsigned long long)total * die / 8) + (blockIdx.x >> 3);
  }

  struct Tile {
    int n0, n_here, m_here, first, expert, k_end;  // m_here 0: there is none
    int begin, sum;                                // DWEIGHTS: the part's first row, and its place among the sums
  };
  // the next tile of this workgroup
  auto locate = [&]() {
    Tile r = {0, 0, 0, 0, 0, 0, 0, -1};
    for (; tile < tiles_end && r.m_here <= 0; tile += gridDim.x >> 3) {
      const unsigned band = (unsigned)a.band * a.n_tiles, m0 = tile / band * a.band;
      const unsigned high = m_tiles - m0 < (unsigned)a.band ? m_tiles - m0 : a.band;
      const unsigned in = tile % band;
      const int number = (int)(m0 + in % high), n_tile = (int)(in / high);
      r.n0 = n_tile * BN, r.n_here = a.n - r.n0 < BN ? a.n - r.n0 : BN;
      r.k_end = a.k;
      if constexpr (KIND == DWEIGHTS) {
        const int tiles = (a.k + BM - 1) / BM;
        r.first = number % tiles * BM;
        PartOfRows part;
        if (in_parts) {
          if (!part_of_rows(a.offsets, a.experts, a.rows, a.part, number / tiles, part)) continue;
        } else {
          const int begin = a.offsets[number / tiles];
          part = {number / tiles, begin, a.offsets[number / tiles + 1] - begin, -1};
        }
        r.expert = __builtin_amdgcn_readfirstlane(part.expert), r.k_end = part.rows;
        r.begin = __builtin_amdgcn_readfirstlane(part.first), r.sum = __builtin_amdgcn_readfirstlane(part.sum);
        r.m_here = a.k - r.first < BM ? a.k - r.first : BM;
      } else if (ragged) {
        if (listed)
          listed_tile<BM>(table, a.offsets, a.experts, a.rows, number, r.expert, r.first, r.m_here);
        else
          ragged_tile(a.offsets, a.experts, a.rows, BM, number, r.expert, r.first, r.m_here);
        if (r.expert == a.experts) r.k_end = 0, r.expert = 0;  // rows without an expert: zeros
      } else {
        r.first = number * BM, r.m_here = a.rows - r.first < BM ? a.rows - r.first : BM;
      }
    }
    r.m_here = __builtin_amdgcn_readfirstlane(r.m_here > 0 ? r.m_here : 0);
    r.first = __builtin_amdgcn_readfirstlane(r.first);
    r.k_end = __builtin_amdgcn_readfirstlane(r.k_end);
    return r;
  };
  // x's rows of a tile, for the lanes that load them later
  auto order_of = [&](const Tile &r) -> int {
    const int m = (int)threadIdx.x % BM;
    return GATHER && r.m_here > 0 ? a.order[r.first + (m < r.m_here ? m : r.m_here - 1)] : 0;
  };
  unsigned rows_put = 0, rows_in = BM;  // which of the two is written next, and which is read
  auto put_order = [&](int slot) {
    if (GATHER && threadIdx.x < BM) gathered[rows_put + threadIdx.x] = (unsigned)(slot / a.top_k);
    rows_put ^= BM;
  };

  // ---- what is loaded
  // Where a lane's pieces lie behind a stage's start. No piece is clamped: what lies behind the operand's last byte of
  // the stage is not read, and a piece of a row or column that does not exist is multiplied into what is not stored, or
  // masked. From one of a lane's pieces to its next, THREADS slots on, are so many rows or k, turned alike.
  // (float32 in columns: eight k on, every second is turned the other way.)
  constexpr int ODD = SIZE == 4 ? 2 : 1;
  unsigned x_off[ODD], w_off[ODD];
  const unsigned x_next = (unsigned)((XC ? THREADS / X::Tile::PER_K : THREADS / 8) * a.x_stride);
  const unsigned w_next = (unsigned)((WC ? THREADS / W::Tile::PER_K : THREADS / 8) * a.w_stride);
#pragma unroll
  for (int i = 0; i < ODD; ++i) {
    int r, k;
    W::Tile::place(i * THREADS + threadIdx.x, r, k);
    w_off[i] = (WC ? (unsigned)(k * a.w_stride) + r * SIZE : (unsigned)(r * a.w_stride) + k * SIZE) - i * w_next;
    X::Tile::place(i * THREADS + threadIdx.x, r, k);
    x_off[i] = GATHER ? k * SIZE
                      : (XC ? (unsigned)(k * a.x_stride) + r * SIZE : (unsigned)(r * a.x_stride) + k * SIZE) - i * x_next;
  }
  const size_t x_step = XC ? KS * a.x_stride : 128, w_step = WC ? KS * a.w_stride : 128;
  Tile in;  // the tile that is loaded
  const char *in_x = nullptr, *in_w = nullptr, *in_s = nullptr;
  unsigned in_s_size = 0;
  int in_left = 0, in_stages = 0, in_stage = 0;  // k and stages that are left, and the number of the next one
  auto enter = [&](const Tile &r) {
    in = r;
    in_x = a.x, in_w = a.w;
    if constexpr (KIND == DWEIGHTS) {
      in_x += (size_t)r.begin * a.x_stride + (size_t)r.first * SIZE;
      in_w += (size_t)r.begin * a.w_stride + (size_t)r.n0 * SIZE;
    } else {
      if (!GATHER) in_x += (size_t)r.first * a.x_stride;
      in_w += (size_t)r.expert * a.w_expert + (WC ? (size_t)r.n0 * SIZE : (size_t)r.n0 * a.w_stride);
    }
    in_x = same_in_all(in_x), in_w = same_in_all(in_w);
    settled(in_x, in_w);
    in_left = r.k_end, in_stages = r.m_here ? stages_of(r.k_end) : 0x7fffffff, in_stage = 0;
    if (r.m_here == 0) in_left = 0;
    rows_in ^= BM;
    if constexpr (FOUR) {
      const bool of_x = wave * 64 < BM;
      const size_t row = of_x ? (GATHER ? 0 : (size_t)r.first) : (size_t)r.expert * a.n + r.n0;
      const unsigned rows = of_x ? (GATHER ? (unsigned)(a.x_bytes / a.x_stride) : (unsigned)r.m_here) : (unsigned)r.n_here;
      in_s = same_in_all((const char *)(of_x ? a.x_scales : a.w_scales) + row * a.scales_stride);
      in_s_size = __builtin_amdgcn_readfirstlane((rows - 1) * (unsigned)a.scales_stride + 16);
      settled(in_s, in_s_size);
    }
  };
  unsigned x_size = 0, w_size = 0;
  auto whole = [](int elements) { return (unsigned)(elements * SIZE + 3) & ~3u; };  // bytes of their words
  auto size_up = [&]() {  // of the stage that is loaded now
    const int k_here = in_left < KS ? in_left : KS;
    x_size = k_here <= 0 ? 0
             : GATHER    ? (unsigned)(a.x_bytes - (size_t)in_stage * 128)
             : XC        ? (unsigned)((k_here - 1) * a.x_stride) + whole(in.m_here)
                         : (unsigned)((in.m_here - 1) * a.x_stride) + whole(k_here);
    w_size = k_here <= 0 ? 0
             : WC        ? (unsigned)((k_here - 1) * a.w_stride) + whole(in.n_here)
                         : (unsigned)((in.n_here - 1) * a.w_stride) + whole(k_here);
  };
  unsigned buffer = 0;  // of the stage that is loaded now: 0 or STAGE
  unsigned row_off[GATHER ? X::P : 1];
  auto find_rows = [&]() {  // (kept over a stage only, for want of registers)
    if constexpr (GATHER) {
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));
#pragma unroll
      for (int i = 0; i < X::P; ++i) row_off[i] = gathered[rows_in + i * (THREADS / 8) + tid / 8] * (unsigned)a.x_stride;
    }
  };
  auto load_one = [&](int i) {
    if (i < X::P)
      to_lds_16(buffer_of(in_x, x_size), x_off[i % ODD] + (GATHER ? row_off[GATHER ? i : 0] : i * x_next),
                to + buffer + i * THREADS * 16);
    else
      to_lds_16(buffer_of(in_w, w_size), w_off[(i - X::P) % ODD] + (i - X::P) * w_next,
                to + buffer + BM * 128 + (i - X::P) * THREADS * 16);
  };
  unsigned scales_in = 0;  // 0 or SCALES
  auto load_scales = [&]() {  // of this stage and the next, 512 columns, at every even stage of a tile
    if constexpr (FOUR) {
      if (!(in_stage & 1)) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const unsigned row = GATHER && wave * 64 < BM ? gathered[rows_in + tid % BM] : tid % BM;
        to_lds_16(buffer_of(in_s + (size_t)in_stage * 8, in_left > 0 ? in_s_size : 0), row * (unsigned)a.scales_stride,
                  to + 2 * STAGE + scales_in);
        scales_in ^= SCALES;
      }
    }
  };
  auto loaded = [&]() {
    in_x += x_step, in_w += w_step, in_left -= KS, ++in_stage, buffer ^= STAGE;
  };

  // ---- what is multiplied
  f32x4 acc[FM][FN];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  X fx;
  W fw;
  fx.init(base, threadIdx.x & 63, wm * FM);
  fw.init(base + BM * 128, threadIdx.x & 63, wn * FN);
  unsigned s_at = base + 2 * STAGE + (threadIdx.x & 15) * 16 + (threadIdx.x & 48) / 4;

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
  unsigned sx[FOUR ? FM : 1], sw[FOUR ? FN : 1];
  auto read_scales = [&](int t) {  // words of the four steps of two stages: their low halves count
    if constexpr (FOUR) {
      if (t & 1) {
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] >>= 16;
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] >>= 16;
      } else {
#pragma unroll
        for (int j = 0; j < FN; ++j) sw[j] = lds_read_4(s_at + BM * 16 + (wn * FN + j) * 256);
#pragma unroll
        for (int i = 0; i < FM; ++i) sx[i] = lds_read_4(s_at + (wm * FM + i) * 256);
      }
    }
  };
  auto multiply_one = [&](auto step, int q) {
    constexpr int S = decltype(step)::value;
    const int i = q / FN, j = q % FN;
    if constexpr (FOUR)
      mfma_four<S>(acc[i][j], f[S].w[j], f[S].x[i], sw[j], sx[i]);
    else
      mfma_piece(acc[i][j], f[S].w[j], f[S].x[i], Tag<T>());
  };
  // A step's products, with the LDS reads of the next step spread between the first 3/4 of them and `loads` loads between
  // all. (A load takes its turn in the CU's address unit; a wavefront that has to wait for that issues nothing else.)
  auto multiply = [&](auto step, auto loads, auto load_it) {
    constexpr int S = decltype(step)::value, R = FM + FN, L = decltype(loads)::value, Q = FM * FN, SPAN = Q * 3 / 4;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r * SPAN / R == q) read_one(Int<1 - S>(), r);
#pragma unroll
      for (int l = 0; l < L; ++l)
        if (l * Q / (L ? L : 1) == q) load_it(l);
      multiply_one(step, q);
      __builtin_amdgcn_sched_barrier(0);
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
  // A step that reaches behind the last k (`left` are there): what lies there is no part of the sum, and may be anything.
  auto mask = [&](auto step, int left) {
    constexpr int S = decltype(step)::value;
    left -= S * (KS / 2) + EPP * ((threadIdx.x & 63) >> 4);
    const u32x4 keep = first_of<T>(left);
#pragma unroll
    for (int i = 0; i < FM; ++i) f[S].x[i] &= keep;
#pragma unroll
    for (int j = 0; j < FN; ++j) f[S].w[j] &= keep;
  };

  Tile now = locate();  // the tile that is multiplied
  if (now.m_here == 0) return;
  put_order(order_of(now));
  __syncthreads();
  enter(now);
  for (int s = 0; s < 2; ++s) {  // (a tile has two stages at least)
    size_up();
    find_rows();
#pragma unroll
    for (int i = 0; i < X::P + W::P; ++i) load_one(i);
    load_scales();
    loaded();
    if (s == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  Tile ahead = locate();
  __syncthreads();
  put_order(order_of(ahead));
  clear();
#pragma unroll
  for (int r = 0; r < FM + FN; ++r) read_one(Int<0>(), r);
  read_scales(0);
  for (int t = 0, left = now.k_end;;) {
    if (!FOUR && left < KS) mask(Int<0>(), left);
    multiply(Int<0>(), Int<0>(), [](int) {});
    meet();
    if (in_stage == in_stages) enter(ahead);
    size_up();
    find_rows();
    if (!FOUR && left < KS) mask(Int<1>(), left);
    fx.swap(STAGE), fw.swap(STAGE);
    multiply(Int<1>(), Int<X::P + W::P>(), load_one);
    load_scales();
    loaded();
    ++t, left -= KS;
    if (FOUR && !(t & 1)) s_at = scales_swapped(s_at, SCALES, base + 2 * STAGE);
    if (t == stages_of(now.k_end)) {
      if (FOUR) {
        if (t & 1) s_at = scales_swapped(s_at, SCALES, base + 2 * STAGE);
        if (now.k_end == 0) clear();
      }
      // `in` is the tile that comes now; the one after it is looked for while this one goes out
      const Tile next = in;
      ahead = locate();
      const int slot = order_of(ahead);
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (what follows from it is not kept over the stages)
      if (KIND == DWEIGHTS && now.sum >= 0)
        store_tile<float, FM, FN>(tid & 63, acc, a.sums + (size_t)now.sum * a.c_expert + (size_t)now.first * a.c_stride + now.n0,
                                  a.c_stride, wm * FM * 16, wn * FN * 16, now.m_here, now.n_here);
      else
        store_tile<OUT, FM, FN>(tid & 63, acc,
                                static_cast<OUT *>(a.c) + (KIND == DWEIGHTS ? (size_t)now.expert * a.c_expert : 0) +
                                    (size_t)now.first * a.c_stride + now.n0,
                                a.c_stride, wm * FM * 16, wn * FN * 16, now.m_here, now.n_here);
      put_order(slot);
      now = next;
      if (now.m_here == 0) break;
      t = 0, left = now.k_end;
      clear();
    }
    read_scales(t);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads that read nothing end before the LDS is another's)
}

template <typename ELEMENT, typename OUT, Kind KIND, bool GATHER, int BM, int BN, int WM, int WN>
int launch_pipe(PipeArgs &a, hipStream_t stream) {
  const size_t m_tiles = KIND == DWEIGHTS ? (a.part < a.rows ? ragged_tiles(a.experts, a.rows, a.part) : (size_t)a.experts) *
                                                ((a.k + BM - 1) / BM)
                         : a.experts      ? ragged_tiles(a.experts, a.rows, BM)
                                          : ((size_t)a.rows + BM - 1) / BM;
  a.m_tiles = (int)m_tiles, a.n_tiles = (a.n + BN - 1) / BN;
  // (as many tiles of m beside each other as make the operands that a chiplet's workgroups read at once few: 8192^3 in
  // bfloat16 912 us, with bands of one tile 985, of 64 1150)
  a.band = a.n_tiles >= 8 ? 4 : a.n_tiles >= 4 ? 8 : 16;
  const size_t tiles = m_tiles * a.n_tiles;
  if (m_tiles > (size_t)INT_MAX || tiles > (size_t)INT_MAX) return H2O4GPU_KMEANS_EARG;
  const size_t lds =
      (BM + BN) * (256 + (__is_same(ELEMENT, Four) ? 32 : 0)) + (GATHER ? BM * 8 : 0) + (PIPE_TABLE + 2 + WM * WN) * 4;
  const auto kernel = pipe_kernel<ELEMENT, OUT, KIND, GATHER, BM, BN, WM, WN>;
  KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds));
  constexpr size_t WORKGROUPS = BM + BN == 512 ? 256 : 512;  // as many as the CUs' LDS allows
  const size_t blocks = tiles < WORKGROUPS ? (tiles + 7) / 8 * 8 : WORKGROUPS;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(WM * WN * 64), lds, stream, a);
  return launched();
}

// In tiles of 256 x 256, or of 128 x 128, of which a CU holds two.
template <typename ELEMENT, typename OUT, Kind KIND, bool GATHER>
int launch_large(PipeArgs &a, Way way, hipStream_t stream) {
  if (way == TILES_256) return launch_pipe<ELEMENT, OUT, KIND, GATHER, 256, 256, 2, 4>(a, stream);
  return launch_pipe<ELEMENT, OUT, KIND, GATHER, 128, 128, 2, 2>(a, stream);
}

}  // namespace kmhip
