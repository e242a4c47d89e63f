// Products of few rows: the matrices are read once, straight into the registers of the matrix instructions' operand, and
// that is what bounds them. A wavefront has 16 NB rows of a matrix and MB blocks of 16 rows of x; `share` wavefronts of a
// workgroup (a power of two) share the columns and add up their sums in LDS, the others have other rows of the matrix.
// 8 experts' 16 rows with 7168 x 4096, bfloat16 (470 MB of matrices), take 78 us, 6.0 TB/s, the rows' gradient 85; 64
// experts' 256 rows with 2048 x 2048 104 and 100 us; 16 rows times 8192 x 8192 in 4 bits (36 MB) 12, one row 8.
#pragma once

#include "product_pipe.h"

namespace kmhip {

struct ThinArgs {
  const char *x, *w;
  const unsigned char *x_scales, *w_scales;            // Four only, rows of `scales_stride` bytes
  void *c;
  size_t x_stride, w_stride, w_expert, scales_stride;  // bytes
  size_t c_stride;                                     // elements
  const int *order, *offsets;                          // as in PipeArgs
  int top_k, experts, rows, n, k;                      // k in elements (Four: in groups of four columns)
  unsigned first_block;
  int halves;          // some row of x or of a matrix begins between words
  int share, n_tiles;  // wavefronts that share columns; workgroups to a block of rows
};

// ALIGNED: every piece lies at a multiple of 16 bytes, and k is whole pieces.
template <typename ELEMENT, typename OUT, int MB, int NB, int WAVES, bool ALIGNED>
__global__ __launch_bounds__(WAVES * 64) void thin_kernel(ThinArgs a) {
  typedef typename PipeElement<ELEMENT>::type T;
  constexpr bool FOUR = __is_same(ELEMENT, Four);
  constexpr int SIZE = (int)sizeof(T), EPP = 16 / SIZE, STEP = 4 * EPP, U = 4;  // k of a step; steps of a turn
  __shared__ f32x4 sums[WAVES][MB * NB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const unsigned block = a.first_block + blockIdx.x;
  const int part = wave & (a.share - 1), row = wave / a.share;
  const int n0 = ((int)(block % (unsigned)a.n_tiles) * (WAVES / a.share) + row) * (16 * NB);
  const int number = (int)(block / (unsigned)a.n_tiles);
  int expert = 0, first = number * (16 * MB), m_here = a.rows - first < 16 * MB ? a.rows - first : 16 * MB, k = a.k;
  if (a.experts) {
    if (!ragged_tile(a.offsets, a.experts, a.rows, 16 * MB, number, expert, first, m_here)) return;
    if (expert == a.experts) k = 0, expert = 0;  // rows without an expert: zeros
  }
  const int n_here = a.n - n0 < 16 * NB ? a.n - n0 : 16 * NB;  // (not positive: nothing to do but to meet the others)
  if (n_here <= 0) k = 0;

  f32x4 acc[MB][NB];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // rows that do not exist are read at the last one that does
  const char *x[MB], *w[NB];
  const unsigned char *xs[FOUR ? MB : 1], *ws[FOUR ? NB : 1];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int p = first + (m * 16 + i < m_here ? m * 16 + i : m_here - 1);
    const size_t row = a.order && k ? (size_t)(a.order[p] / a.top_k) : (size_t)p;
    x[m] = a.x + row * a.x_stride + g * 16;
    if constexpr (FOUR) xs[m] = a.x_scales + row * a.scales_stride + 4 * g;
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int r = n_here <= 0 ? 0 : n0 + (n * 16 + i < n_here ? n * 16 + i : n_here - 1);
    w[n] = a.w + (size_t)expert * a.w_expert + (size_t)r * a.w_stride + g * 16;
    if constexpr (FOUR) ws[n] = a.w_scales + ((size_t)expert * a.n + r) * a.scales_stride + 4 * g;
  }
  const int turns = (k + U * STEP - 1) / (U * STEP);
  // a wavefront's turns lie side by side
  const int each = (turns + a.share - 1) / a.share, begin = part * each, end = begin + each < turns ? begin + each : turns;
  u32x4 fx[U][MB], fw[U][NB];
  unsigned sx[FOUR ? MB : 1], sw[FOUR ? NB : 1];
  auto load = [&](int t) {
    auto all = [&](bool halves) __attribute__((always_inline)) {  // (no branches: all loads are on their way at once)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t at = ((size_t)t * U + u) * 64;
#pragma unroll
        for (int n = 0; n < NB; ++n)
          fw[u][n] = ALIGNED ? *reinterpret_cast<const u32x4 *>(w[n] + at)
                             : load_whole(reinterpret_cast<const T *>(w[n] + at), halves);
#pragma unroll
        for (int m = 0; m < MB; ++m)
          fx[u][m] = ALIGNED ? *reinterpret_cast<const u32x4 *>(x[m] + at)
                             : load_whole(reinterpret_cast<const T *>(x[m] + at), halves);
      }
    };
    if ((t + 1) * (U * STEP) <= k) {
      if (!ALIGNED && a.halves)
        all(true);
      else
        all(false);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t at = ((size_t)t * U + u) * 64;
        const int left = k - ((t * U + u) * STEP + g * EPP);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if constexpr (ALIGNED)
            fw[u][n] = left > 0 ? *reinterpret_cast<const u32x4 *>(w[n] + at) : u32x4{0, 0, 0, 0};
          else
            fw[u][n] = load_piece(reinterpret_cast<const T *>(w[n] + at), left);
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
          if constexpr (ALIGNED)
            fx[u][m] = left > 0 ? *reinterpret_cast<const u32x4 *>(x[m] + at) : u32x4{0, 0, 0, 0};
          else
            fx[u][m] = load_piece(reinterpret_cast<const T *>(x[m] + at), left);
        }
      }
    }
    if constexpr (FOUR) {
#pragma unroll
      for (int n = 0; n < NB; ++n) sw[n] = *reinterpret_cast<const unsigned *>(ws[n] + (size_t)t * 16);
#pragma unroll
      for (int m = 0; m < MB; ++m) sx[m] = *reinterpret_cast<const unsigned *>(xs[m] + (size_t)t * 16);
    }
  };
  for (int t = begin; t < end; ++t) {
    load(t);
    auto step = [&](auto number) {
      constexpr int S = decltype(number)::value;
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if constexpr (FOUR)
            mfma_four<S>(acc[m][n], fw[S][n], fx[S][m], sw[n], sx[m]);
          else
            mfma_piece(acc[m][n], fw[S][n], fx[S][m], Tag<T>());
        }
    };
    step(Int<0>());
    step(Int<1>());
    step(Int<2>());
    step(Int<3>());
  }
  auto store = [&](int b, f32x4 s) {
    const int m = b / NB * 16 + i, n = b % NB * 16 + 4 * g;
    if (m < m_here) store_four(static_cast<OUT *>(a.c) + (size_t)(first + m) * a.c_stride + n0 + n, s, n_here - n);
  };
  if (a.share == 1) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) store(m * NB + n, acc[m][n]);
    return;
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n) sums[wave][m * NB + n][lane] = acc[m][n];
  __syncthreads();
  for (int b = part; b < MB * NB; b += a.share) {
    f32x4 s = sums[wave - part][b][lane];
    for (int v = 1; v < a.share; ++v) s += sums[wave - part + v][b][lane];
    store(b, s);
  }
}

// One matrix in 4 bits, x of 17 to 64 rows and at most 8192 columns: a workgroup keeps its part of x, which it would read
// from L2 for every 32 rows of the matrix (33 rows of 8190 times 11003, with what makes 4 bits of x: 29 us that way and 21
// this, of which the matrix takes 10), and takes 16 rows after others, the next of which are on their way while these are
// multiplied.
template <typename OUT, int MB>
__global__ __launch_bounds__(512) void kept_kernel(ThinArgs a) {
  constexpr int WAVES = 8, U = 4, TURNS = 2;
  __shared__ f32x4 sums[2][WAVES][MB][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int steps = (a.k + 31) / 32;  // of 64 bytes a row
  const int first = wave * TURNS * U;  // of this wavefront's
  u32x4 fx[TURNS][U][MB], fw[2][TURNS][U];
  unsigned sx[TURNS][MB], sw[2][TURNS];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const size_t row = m * 16 + i < a.rows ? m * 16 + i : a.rows - 1;
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = first + t * U + u;
        fx[t][u][m] = s < steps ? *reinterpret_cast<const u32x4 *>(a.x + row * a.x_stride + (size_t)s * 64 + g * 16)
                                : u32x4{0, 0, 0, 0};
      }
      sx[t][m] = first + t * U < steps ? *reinterpret_cast<const unsigned *>(a.x_scales + row * a.scales_stride +
                                                                            (size_t)(wave * TURNS + t) * 16 + 4 * g)
                                       : 0;
    }
  }
  auto load = [&](auto b, int tile) {
    constexpr int B = decltype(b)::value;
    const int n = tile * 16 + i;
    const size_t row = n < a.n ? n : a.n - 1;
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = first + t * U + u;
        if (s < steps) fw[B][t][u] = *reinterpret_cast<const u32x4 *>(a.w + row * a.w_stride + (size_t)s * 64 + g * 16);
      }
      if (first + t * U < steps)
        sw[B][t] = *reinterpret_cast<const unsigned *>(a.w_scales + row * a.scales_stride + (size_t)(wave * TURNS + t) * 16 +
                                                       4 * g);
    }
  };
  auto multiply = [&](auto b, int tile) {
    constexpr int B = decltype(b)::value;
    f32x4 acc[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
      auto step = [&](auto number) {
        constexpr int S = decltype(number)::value;
        if (first + t * U + S < steps) {
#pragma unroll
          for (int m = 0; m < MB; ++m) mfma_four<S>(acc[m], fw[B][t][S], fx[t][S][m], sw[B][t], sx[t][m]);
        }
      };
      step(Int<0>());
      step(Int<1>());
      step(Int<2>());
      step(Int<3>());
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) sums[B][wave][m][lane] = acc[m];
    __syncthreads();
    if (wave < MB) {
      f32x4 s = sums[B][0][wave][lane];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) s += sums[B][v][wave][lane];
      const int m = wave * 16 + i, n = tile * 16 + 4 * g;
      if (m < a.rows) store_four(static_cast<OUT *>(a.c) + (size_t)m * a.c_stride + n, s, a.n - n);
    }
  };
  int tile = blockIdx.x;
  load(Int<0>(), tile);
  for (;;) {
    const int next = tile + (int)gridDim.x, after = next + (int)gridDim.x;
    if (next < a.n_tiles) load(Int<1>(), next);
    multiply(Int<0>(), tile);
    if (next >= a.n_tiles) break;
    if (after < a.n_tiles) load(Int<0>(), after);
    multiply(Int<1>(), next);
    if (after >= a.n_tiles) break;
    tile = after;
  }
}

template <typename OUT>
int launch_kept(ThinArgs &a, hipStream_t stream) {
  a.n_tiles = (a.n + 15) / 16;
  const unsigned blocks = a.n_tiles < 256 ? a.n_tiles : 256;
  auto launch = [&](auto mb) {
    hipLaunchKernelGGL((kept_kernel<OUT, decltype(mb)::value>), dim3(blocks), dim3(512), 0, stream, a);
    return launched();
  };
  return a.rows <= 32 ? launch(Int<2>()) : a.rows <= 48 ? launch(Int<3>()) : launch(Int<4>());
}

template <typename ELEMENT, typename OUT, bool ALIGNED>
int launch_thin(ThinArgs &a, hipStream_t stream) {
  const int each = a.experts ? a.rows / a.experts : a.rows;  // rows of an expert, on average
  auto launch = [&](auto mb, auto nb) {
    constexpr int MB = decltype(mb)::value, NB = decltype(nb)::value, WAVES = 8;
    const size_t m_tiles =
        a.experts ? ragged_tiles(a.experts, a.rows, 16 * MB) : ((size_t)a.rows + 16 * MB - 1) / (16 * MB);
    // a wavefront for each turn of a row, up to the workgroup's
    constexpr int TURN = 4 * 4 * (16 / (int)sizeof(typename PipeElement<ELEMENT>::type));
    const int turns = (a.k + TURN - 1) / TURN;
    a.share = turns > 4 ? 8 : turns > 2 ? 4 : turns > 1 ? 2 : 1;
    a.n_tiles = (a.n + 16 * NB * (WAVES / a.share) - 1) / (16 * NB * (WAVES / a.share));
    return in_launches(m_tiles * a.n_tiles, [&](unsigned first, unsigned blocks) {
      a.first_block = first;
      hipLaunchKernelGGL((thin_kernel<ELEMENT, OUT, MB, NB, WAVES, ALIGNED>), dim3(blocks), dim3(WAVES * 64), 0, stream, a);
      return launched();
    });
  };
  if (each <= 16) return launch(Int<1>(), Int<1>());
  if (each <= 32) return launch(Int<2>(), Int<2>());
  if (each <= 48) return launch(Int<3>(), Int<2>());
  return launch(Int<4>(), Int<2>());
}

// thin_kernel's product where the matrix lies with n side by side (W^T dy): a lane loads 16 bytes, EPP columns, of some
// k's of its own; element b of all of them is its fragment of a block of 16 columns, EPP apart, so that a wavefront has 16
// EPP columns. What comes out for a lane and a j, block by block, is EPP columns side by side again.
template <typename T, bool HALVES, int MB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void thin_columns_kernel(ThinArgs a) {
  constexpr int EPP = 16 / (int)sizeof(T), STEP = 4 * EPP, TURN = 32, U = TURN / STEP;  // k of a turn
  __shared__ f32x4 sums[WAVES][MB * EPP][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const unsigned block = a.first_block + blockIdx.x;
  const int part = wave & (a.share - 1);
  const int n0 = ((int)(block % (unsigned)a.n_tiles) * (WAVES / a.share) + wave / a.share) * (16 * EPP);
  int expert, first, m_here, k = a.k;
  if (!ragged_tile(a.offsets, a.experts, a.rows, 16 * MB, (int)(block / (unsigned)a.n_tiles), expert, first, m_here)) return;
  if (expert == a.experts) k = 0, expert = 0;  // rows without an expert: zeros
  if (a.n <= n0) k = 0;

  f32x4 acc[MB][EPP];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int b = 0; b < EPP; ++b) acc[m][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T *x[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m)
    x[m] = reinterpret_cast<const T *>(a.x + (size_t)(first + (m * 16 + i < m_here ? m * 16 + i : m_here - 1)) * a.x_stride);
  const size_t w = (size_t)(a.w + (size_t)expert * a.w_expert + (size_t)n0 * sizeof(T));
  const unsigned behind = (unsigned)(w & 3);  // of the first word
  const int n_here = a.n - n0 < 16 * EPP ? a.n - n0 : 16 * EPP;
  const int turns = (k + TURN - 1) / TURN, each = (turns + a.share - 1) / a.share;
  const int begin = part * each, end = begin + each < turns ? begin + each : turns;
  struct Turn {
    u32x4 x[U][MB], w[U][EPP];
    unsigned last[HALVES ? U : 1][EPP];
  } turn[2];
  auto load = [&](Turn &f, int t) __attribute__((always_inline)) {
    const char *from = same_in_all((const char *)(w - behind + (size_t)t * TURN * a.w_stride));
    const int here = k - t * TURN < TURN ? k - t * TURN : TURN;
    const unsigned size = ((unsigned)((here - 1) * a.w_stride + (size_t)n_here * sizeof(T)) + behind + 3) & ~3u;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int r = 0; r < EPP; ++r) {
        const unsigned at = (unsigned)((u * STEP + EPP * g + r) * a.w_stride) + EPP * i * (unsigned)sizeof(T) + behind;
        f.w[u][r] = buffer_words(from, size, HALVES ? at & ~3u : at);
        if (HALVES) f.last[u][r] = buffer_word(from, size, (at + 14) & ~3u);
      }
    }
    // (the last k's of a row of x one by one: behind it may be nothing)
    if ((t + 1) * TURN <= k) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MB; ++m) f.x[u][m] = load_whole(x[m] + t * TURN + u * STEP + EPP * g, HALVES);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MB; ++m)
          f.x[u][m] = load_piece(x[m] + t * TURN + u * STEP + EPP * g, k - (t * TURN + u * STEP + EPP * g));
    }
  };
  auto multiply = [&](Turn &f, int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k0 = t * TURN + u * STEP + EPP * g;
#pragma unroll
      for (int r = 0; r < EPP; ++r) {
        if (HALVES)
          f.w[u][r] = shifted(f.w[u][r], f.last[u][r],
                              (unsigned)((u * STEP + EPP * g + r) * a.w_stride + EPP * i * sizeof(T) + behind) & 2);
        if (k0 + r >= k) f.w[u][r] = u32x4{0, 0, 0, 0};  // (whatever lies there)
      }
#pragma unroll
      for (int b = 0; b < EPP; ++b) {
        u32x4 v;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          if constexpr (sizeof(T) == 4)
            v[d] = f.w[u][d][b];
          else
            v[d] = __builtin_amdgcn_perm(f.w[u][2 * d + 1][b / 2], f.w[u][2 * d][b / 2], b & 1 ? 0x07060302u : 0x05040100u);
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) mfma_piece(acc[m][b], v, f.x[u][m], Tag<T>());
      }
    }
  };
  if (begin < end) {
    load(turn[0], begin);
    for (int t = begin;; t += 2) {  // a turn is on its way while one is multiplied
      if (t + 1 < end) load(turn[1], t + 1);
      multiply(turn[0], t);
      if (t + 1 >= end) break;
      if (t + 2 < end) load(turn[0], t + 2);
      multiply(turn[1], t + 1);
      if (t + 2 >= end) break;
    }
  }
  auto store = [&](int m, int j, const float (&s)[EPP]) {
    const int n = n0 + EPP * (4 * g + j), valid = a.n - n;
    if (m * 16 + i >= m_here || valid <= 0) return;
    T *to = static_cast<T *>(a.c) + (size_t)(first + m * 16 + i) * a.c_stride + n;
    typename Beside<T, EPP>::vector p;
#pragma unroll
    for (int b = 0; b < EPP; ++b) p[b] = (T)s[b];
    if (valid >= EPP) {
      store_beside<T, EPP>(to, p);
    } else {
#pragma unroll
      for (int b = 0; b < EPP - 1; ++b)
        if (b < valid) to[b] = p[b];
    }
  };
  if (a.share > 1) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int b = 0; b < EPP; ++b) sums[wave][m * EPP + b][lane] = acc[m][b];
    __syncthreads();
    for (int q = part; q < MB * 4; q += a.share) {
      float s[EPP];
#pragma unroll
      for (int b = 0; b < EPP; ++b) s[b] = sums[wave - part][q / 4 * EPP + b][lane][q % 4];
      for (int p = 1; p < a.share; ++p)
#pragma unroll
        for (int b = 0; b < EPP; ++b) s[b] += sums[wave - part + p][q / 4 * EPP + b][lane][q % 4];
      store(q / 4, q % 4, s);
    }
  } else {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float s[EPP];
#pragma unroll
        for (int b = 0; b < EPP; ++b) s[b] = acc[m][b][j];
        store(m, j, s);
      }
  }
}

template <typename T>
int launch_thin_columns(ThinArgs &a, hipStream_t stream) {
  auto launch = [&](auto mb, auto waves) {
    constexpr int MB = decltype(mb)::value, WAVES = decltype(waves)::value, COLS = 16 * (16 / (int)sizeof(T));
    const int turns = (a.k + 31) / 32;
    a.share = turns >= WAVES ? WAVES : turns > 2 ? 4 : turns > 1 ? 2 : 1;
    a.n_tiles = (a.n + COLS * (WAVES / a.share) - 1) / (COLS * (WAVES / a.share));
    return in_launches(ragged_tiles(a.experts, a.rows, 16 * MB) * a.n_tiles, [&](unsigned first, unsigned blocks) {
      a.first_block = first;
      if (sizeof(T) == 2 && a.halves)
        hipLaunchKernelGGL((thin_columns_kernel<T, sizeof(T) == 2, MB, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, stream, a);
      else
        hipLaunchKernelGGL((thin_columns_kernel<T, false, MB, WAVES>), dim3(blocks), dim3(WAVES * 64), 0, stream, a);
      return launched();
    });
  };
  return a.rows / a.experts <= 16 ? launch(Int<1>(), Int<8>()) : launch(Int<2>(), Int<4>());
}

}  // namespace kmhip
