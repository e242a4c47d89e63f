// Expert layers: the choice of a row's experts, the order of rows by expert, and rows sent out and
// joined again, with their gradients.
#include "experts_common.h"

namespace kmhip {

static const int WAVE = 64;

// Workgroups of a launch whose kernel walks its rows with the grid's stride: a grid has fewer than
// 2^32 threads.
static unsigned grid_of(size_t wanted) { return (unsigned)(wanted < (1u << 22) ? wanted : (1u << 22)); }

// ---------------------------------------------------------------------------
// route
// ---------------------------------------------------------------------------

// A score as a key whose largest value is the best; NaN as the worst.
template <bool LARGEST>
__device__ __forceinline__ float score_key(float s) {
  const float k = LARGEST ? s : -s;
  return k == k ? k : -__builtin_huge_valf();
}

// exp(scale * (k - best)), where the difference of two equal infinities is no difference, nor is any at scale 0.
__device__ __forceinline__ float softmax_term(float k, float best, float scale) {
  return k == best || scale == 0.f ? 1.0f : expf(scale * (k - best));
}

// The same as a term of a sum over all. Its exponent x is a product of two rounded factors and rounded itself, so
// that the term is off by up to 1.5 |x| 2^-23 of it: 0.6 * 2^-23 of the largest one (1), 1.5 ln(E) 2^-23 of the sum.
// scale2: scale * log2(e), of which exp2 is one instruction.
__device__ __forceinline__ float summed_term(float k, float best, float scale2) {
  return k == best || scale2 == 0.f ? 1.0f : __builtin_amdgcn_exp2f(scale2 * (k - best));
}
static const float LOG2E = 1.44269504088896341f;

// The same where it is a result's factor (the gradient of a score that is not chosen, whose own size counts), in a few
// instructions: exp2 has the rounded x log2(e), and a product what that is off by. Terms below 2^-126 are 0.
__device__ __forceinline__ float other_term(float k, float best, float scale) {
  if (k == best || scale == 0.f) return 1.0f;
  const float high = 1.44269504f, low = 1.92596299e-8f;  // log2(e) is their sum
  const float x = fmaxf(scale * (k - best), -200.f), y = x * high;
  const float p = __builtin_amdgcn_exp2f(y), rest = fmaf(x, low, fmaf(x, high, -y));
  return fmaf(p, rest * 0.693147181f, p);
}

__device__ __forceinline__ bool comes_before(float ka, int ia, float kb, int ib) {
  return ka > kb || (ka == kb && ia < ib);
}

// One wavefront a row, any strides, any number of experts: the best entry behind the last one
// chosen, top_k times over the row.
template <typename T, bool LARGEST, bool ALL>
__global__ __launch_bounds__(256) void route_any_kernel(const T *scores, int64_t rs, int64_t es, int64_t rows, int E,
                                                        int K, float scale, int *experts, float *weights) {
  const int lane = threadIdx.x & 63;
  const float ninf = -__builtin_huge_valf();
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
  const T *s = scores + row * rs;
  float last = __builtin_huge_valf(), top = ninf, sum = 0.f, mine = 0.f;
  int last_i = -1, mine_i = -1;
  for (int j = 0; j < K; j++) {
    float b = ninf;
    int bi = 0x7fffffff;
    for (int e = lane; e < E; e += WAVE) {
      const float k = score_key<LARGEST>((float)s[e * es]);
      if (comes_before(last, last_i, k, e) && k > b) {
        b = k;
        bi = e;
      }
    }
    for (int m = 32; m >= 1; m >>= 1) {
      const float ob = __shfl_xor(b, m, WAVE);
      const int oi = __shfl_xor(bi, m, WAVE);
      if (comes_before(ob, oi, b, bi)) {
        b = ob;
        bi = oi;
      }
    }
    if (b == ninf) break;
    if (j == 0) top = b;
    const float p = softmax_term(b, top, scale);
    if (!ALL) sum += p;
    if (lane == j) {
      mine = p;
      mine_i = bi;
    }
    last = b;
    last_i = bi;
  }
  if (ALL && top != ninf) {
    for (int e = lane; e < E; e += WAVE) {
      const float k = score_key<LARGEST>((float)s[e * es]);
      if (k != ninf) sum += softmax_term(k, top, scale);
    }
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, WAVE);
  }
  if (lane < K) {
    experts[row * K + lane] = mine_i;
    weights[row * K + lane] = mine_i >= 0 ? mine / sum : 0.f;
  }
  }
}

// Lane i's value from lane i ^ 1, i ^ 2, the mirrored lane of its 8 and of its 16, or the lane 16 or 32 further:
// what a reduction over 2, 4, 8, 16, 32 or 64 lanes takes in turn.
template <int STEP>
__device__ __forceinline__ unsigned from_step(unsigned v) {
  if (STEP == 0) return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);   // quad_perm 1 0 3 2
  if (STEP == 1) return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  if (STEP == 2) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);  // row_half_mirror
  if (STEP == 3) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true);  // row_mirror
  const bool low = STEP == 4 ? !(threadIdx.x & 16) : !(threadIdx.x & 32);
  if (STEP == 4) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return low ? s[1] : s[0];
  }
  const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return low ? s[1] : s[0];
}

// A score as a number whose largest is the best: 0 for one that is not available. Zeros of either sign are one.
__device__ __forceinline__ unsigned rank_of(float s, bool largest) {
  const float k = largest ? s : -s;
  const unsigned u = __float_as_uint(k == 0.f ? 0.f : k);
  return k > -__builtin_huge_valf() ? ((int)u < 0 ? ~u : u | 0x80000000u) : 0;
}
__device__ __forceinline__ float key_of(unsigned rank) {
  return __uint_as_float((int)rank < 0 ? rank & 0x7fffffffu : ~rank);
}

// The largest (and the least) of LANES lanes' values, in all of them.
template <int LANES, int STEP = 0>
__device__ __forceinline__ unsigned most_of(unsigned v) {
  if constexpr ((1 << STEP) < LANES) return most_of<LANES, STEP + 1>(max(v, from_step<STEP>(v)));
  return v;
}
template <int LANES, int STEP = 0>
__device__ __forceinline__ unsigned least_of(unsigned v) {
  if constexpr ((1 << STEP) < LANES) return least_of<LANES, STEP + 1>(min(v, from_step<STEP>(v)));
  return v;
}
template <int LANES, int STEP = 0>
__device__ __forceinline__ float sum_of(float v) {
  if constexpr ((1 << STEP) < LANES)
    return sum_of<LANES, STEP + 1>(v + __uint_as_float(from_step<STEP>(__float_as_uint(v))));
  return v;
}

// What a row's kernel compares. A 16-bit score's rank and its expert fit into one number, of which the largest is the
// best with the lowest index; a float's rank fills one by itself (and its expert is looked for).
template <typename T>
struct Key {
  static const bool WITH_EXPERT = false;
  static __device__ __forceinline__ unsigned of(T s, bool largest, unsigned) { return rank_of(s, largest); }
  static __device__ __forceinline__ float score(unsigned key) { return key_of(key); }
};
template <>
struct Key<bfloat16_t> {
  static const bool WITH_EXPERT = true;
  static __device__ __forceinline__ unsigned of(bfloat16_t s, bool largest, unsigned e) {
    const unsigned rank = rank_of((float)s, largest);
    return rank ? (rank & 0xffff0000u) | (0xffff - e) : 0;
  }
  static __device__ __forceinline__ float score(unsigned key) {
    return key_of((int)key < 0 ? key & 0xffff0000u : key | 0xffffu);
  }
};
template <>
struct Key<float16_t> {
  static const bool WITH_EXPERT = true;
  static __device__ __forceinline__ unsigned of(float16_t s, bool largest, unsigned e) {
    const float16_t k = largest ? s : -s;
    const unsigned u = k == (float16_t)0 ? 0 : __builtin_bit_cast(unsigned short, k);
    return (float)k > -__builtin_huge_valf() ? (u & 0x8000 ? 0xffff - u : u | 0x8000) << 16 | (0xffff - e) : 0;
  }
  static __device__ __forceinline__ float score(unsigned key) {
    const unsigned rank = key >> 16;
    return (float)__builtin_bit_cast(float16_t, (unsigned short)(rank & 0x8000 ? rank & 0x7fff : 0xffff - rank));
  }
};

// Rows whose scores lie side by side, at most LANES * NV of them: LANES lanes have a row in registers, W scores in
// a row each at a time. Every round takes the best that is left (a lane's own best, then across the lanes) and
// strikes it out, without a branch. Lane j ends with choice j. What bounds it are the rounds: 16384 rows of 256
// bfloat16, eight chosen of all, take 10 us (40 with the kernel above), reading them 2; 200000 x 100, four: 36 and 8;
// 64000 x 1000 floats, eight of all: 134 and 49.
template <typename T, bool ALL, int LANES, int NV>
__global__ __launch_bounds__(256) void route_rows_kernel(const T *scores, int64_t rs, int64_t rows, int E, int K,
                                                         bool largest, float scale, int *experts, float *weights) {
  constexpr int W = NV < (int)(16 / sizeof(T)) ? NV : (int)(16 / sizeof(T));
  const int lane = threadIdx.x & (LANES - 1);
  const int64_t step = (int64_t)gridDim.x * (256 / LANES);
  for (int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const T *s = scores + row * rs;
    unsigned key[NV];
#pragma unroll
    for (int c = 0; c < NV / W; c++) {
      const int e = (c * LANES + lane) * W;
      struct __attribute__((packed, aligned(sizeof(T)))) Some {
        T v[W];
      } some;
      if (e + W <= E) {
        some = *reinterpret_cast<const Some *>(s + e);
#pragma unroll
        for (int i = 0; i < W; i++) key[c * W + i] = Key<T>::of(some.v[i], largest, e + i);
      } else {
#pragma unroll
        for (int i = 0; i < W; i++) key[c * W + i] = e + i < E ? Key<T>::of(s[e + i], largest, e + i) : 0;
      }
    }
    unsigned mine = 0;
    int mine_e = -1;
    float first = 0.f, total = 0.f;
    for (int j = 0; j < K; j++) {
      unsigned best = key[0];
#pragma unroll
      for (int i = 1; i < NV; i++) best = max(best, key[i]);
      best = most_of<LANES>(best);
      if (best == 0) break;
      if (j == 0) {
        first = Key<T>::score(best);
        if (ALL) {
#pragma unroll
          for (int i = 0; i < NV; i++) total += key[i] ? summed_term(Key<T>::score(key[i]), first, scale * LOG2E) : 0.f;
          total = sum_of<LANES>(total);
        }
      }
      if constexpr (Key<T>::WITH_EXPERT) {
        mine_e = lane == j ? 0xffff - (int)(best & 0xffff) : mine_e;
#pragma unroll
        for (int i = 0; i < NV; i++) key[i] = key[i] == best ? 0 : key[i];
      } else {  // the first of its expert's, and that one struck out
        unsigned at = 1u << 30;
#pragma unroll
        for (int i = NV - 1; i >= 0; i--) at = key[i] == best ? i / W * LANES * W + i % W : at;
        at = least_of<LANES>(at + lane * W);
        mine_e = lane == j ? (int)at : mine_e;
        const unsigned here = at - lane * W;
#pragma unroll
        for (int i = 0; i < NV; i++) key[i] = here == (unsigned)(i / W * LANES * W + i % W) ? 0 : key[i];
      }
      mine = lane == j ? best : mine;
    }
    const float weight = mine ? softmax_term(Key<T>::score(mine), first, scale) : 0.f;
    if (!ALL) total = sum_of<LANES>(weight);
    if (lane < K) {
      experts[row * K + lane] = mine_e;
      weights[row * K + lane] = mine ? weight / total : 0.f;
    }
  }
}

// Scores of one expert side by side (row stride 1, the distances of transform): a lane has a row and walks down
// its experts with its best KT in order. The wavefronts of a workgroup each walk a stretch of
// the experts, and their lists are joined in pairs (a later stretch's equal score stays behind). 1M rows x 64, two
// chosen: 51 us, 5.3 TB/s, what a copy reaches. 1000 x 1000, two of all: 17 (some 10 more with the lists joined one
// after another).
// A sum over all is one lane's over up to 16384 terms, which one after another would be off by up to a quarter of
// 2^-24 a term. Eight are added up in pairs, and what an addition of theirs to the sum rounds away (`over`) goes into
// the next. Terms are against a score `ref` that is less than 1 / scale below the best so far and moves up only when
// it is not: every move rounds the sum, and makes what the moves before it rounded a factor e smaller. (Adding one
// term at a time against the best so far is slower too: 1000 x 1000 20 us, 64000 x 1000 with its gradient 232, not 217.)
template <typename T, bool ALL, int KT>
__global__ __launch_bounds__(1024) void route_columns_kernel(const T *scores, int64_t es, int64_t rows, int E, int K,
                                                             bool largest, float scale, int *experts, float *weights) {
  extern __shared__ float lists[];  // [parts][2 KT + 1][64]: keys, experts, sums over all
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6, parts = blockDim.x >> 6;
  const float ninf = -__builtin_huge_valf(), scale2 = scale * LOG2E;
  const int lo = (int)((int64_t)E * part / parts), hi = (int)((int64_t)E * (part + 1) / parts);
  for (int64_t row0 = (int64_t)blockIdx.x * 64; row0 < rows; row0 += (int64_t)gridDim.x * 64) {
    const int64_t row = row0 + lane < rows ? row0 + lane : rows - 1;
    float key[KT], sum = 0.f, ref = ninf, over = 0.f;
    int id[KT];
#pragma unroll
    for (int j = 0; j < KT; j++) {
      key[j] = ninf;
      id[j] = -1;
    }
    const auto insert = [&](float k, int e) {
#pragma unroll
      for (int j = KT - 1; j >= 0; j--) {
        const bool here = k > key[j], above = j > 0 && k > key[j > 0 ? j - 1 : 0];
        key[j] = above ? key[j > 0 ? j - 1 : 0] : here ? k : key[j];
        id[j] = above ? id[j > 0 ? j - 1 : 0] : here ? e : id[j];
      }
    };
    const T *s = scores + row;
    for (int e0 = lo; e0 < hi; e0 += 8) {
      T v[8];
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = s[(int64_t)(e0 + i < hi ? e0 + i : hi - 1) * es];
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; i++) f[i] = e0 + i < hi ? (largest ? (float)v[i] : -(float)v[i]) : ninf;
      if (ALL) {
        float most = f[0], t[8];
#pragma unroll
        for (int i = 1; i < 8; i++) most = fmaxf(most, f[i]);
        if (scale * (most - ref) > 1.f) {
          const float by = summed_term(ref, most, scale2);
          sum *= by;
          over *= by;
          ref = most;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = f[i] > ninf ? summed_term(f[i], ref, scale2) : 0.f;
        const float add = (((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]))) - over;
        const float next = sum + add;
        over = (next - sum) - add;
        sum = next;
      }
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (f[i] > key[KT - 1]) insert(f[i], e0 + i);
    }
    if (ALL) sum = key[0] > ninf ? (sum - over) * summed_term(ref, key[0], scale2) : 0.f;
    if (parts > 1) {  // (a power of two)
      float *mine = lists + (size_t)part * (2 * KT + 1) * 64 + lane;
      const auto put = [&] {
#pragma unroll
        for (int j = 0; j < KT; j++) {
          mine[2 * j * 64] = key[j];
          mine[(2 * j + 1) * 64] = __int_as_float(id[j]);
        }
        mine[2 * KT * 64] = sum;
      };
      __syncthreads();
      put();
      for (int apart = 1; apart < parts; apart *= 2) {
        __syncthreads();
        if (part & (2 * apart - 1)) continue;
        const float *other = mine + (size_t)apart * (2 * KT + 1) * 64;
        if (ALL) {
          const float top = other[0], its = other[2 * KT * 64];
          if (top > key[0])
            sum = (key[0] > ninf ? sum * summed_term(key[0], top, scale2) : 0.f) + its;
          else if (top > ninf)
            sum += its * summed_term(top, key[0], scale2);
        }
#pragma unroll
        for (int j = 0; j < KT; j++) {
          const float k = other[2 * j * 64];
          if (k > key[KT - 1]) insert(k, __float_as_int(other[(2 * j + 1) * 64]));
        }
        if (2 * apart < parts) put();
      }
      if (part > 0) continue;
    }
    if (row0 + lane >= rows) continue;
    float p[KT], total = 0.f;
#pragma unroll
    for (int j = 0; j < KT; j++) {
      p[j] = j < K && id[j] >= 0 ? softmax_term(key[j], key[0], scale) : 0.f;
      total += p[j];
    }
    if (ALL) total = sum;
#pragma unroll
    for (int j = 0; j < KT; j++)
      if (j < K) {
        experts[row * K + j] = id[j];
        weights[row * K + j] = id[j] >= 0 ? p[j] / total : 0.f;
      }
  }
}

// One wavefront a row, any strides: inner = sum of w g over the chosen, then every expert's gradient, in LDS 1024 at
// a time where the chosen ones' are put in their places.
template <typename T, bool ALL>
__global__ __launch_bounds__(256) void route_backward_kernel(const T *scores, int64_t rs, int64_t es, int64_t rows,
                                                             int E, int K, bool largest, float scale,
                                                             const int *experts, const float *weights,
                                                             const float *dweights, T *dscores, int64_t drs,
                                                             int64_t des) {
  __shared__ float held[4][1024];
  const int lane = threadIdx.x & 63;
  float *mine = held[threadIdx.x >> 6];
  const float sign = largest ? scale : -scale, ninf = -__builtin_huge_valf();
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
    int e_mine = -1;
    float w = 0.f, g = 0.f;
    if (lane < K) {
      e_mine = experts[row * K + lane];
      w = weights[row * K + lane];
      g = e_mine >= 0 ? dweights[row * K + lane] : 0.f;
    }
    const float inner = sum_of<64>(w != 0.f ? w * g : 0.f);
    const int e0 = __builtin_amdgcn_readfirstlane(e_mine);
    const float w0 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(w)));
    float top = 0.f;
    if (ALL && e0 >= 0) top = (largest ? 1.f : -1.f) * (float)scores[row * rs + e0 * es];
    const float own = w != 0.f ? sign * w * (g - inner) : 0.f, rest = ALL && e0 >= 0 ? -sign * w0 * inner : 0.f;
    for (int base = 0; base < E; base += 1024) {
      const int end = E - base < 1024 ? E - base : 1024;
      for (int i = lane; i < end; i += WAVE) {
        float d = 0.f;
        if (ALL && rest != 0.f) {
          const float s = (float)scores[row * rs + (base + i) * es], k = largest ? s : -s;
          const float p = k > ninf ? softmax_term(k, top, scale) : 0.f;
          d = p != 0.f ? rest * p : 0.f;
        }
        mine[i] = d;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (e_mine >= base && e_mine < base + end) mine[e_mine - base] = own;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int i = lane; i < end; i += WAVE) dscores[row * drs + (base + i) * des] = (T)mine[i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// The same of rows whose scores, and gradients, lie side by side: LANES lanes have a row, four experts in a row each
// at a time. 16384 x 256 bfloat16, eight of all: 9 us (11 with the kernel above); 64000 x 1000 floats: 108 (140);
// 500000 x 8 float16, two of all, and the choice itself: 23 us with four lanes, 50 with 16 (136).
template <typename T, bool ALL, int LANES>
__global__ __launch_bounds__(256) void route_backward_rows_kernel(const T *scores, int64_t rs, int64_t rows, int E,
                                                                  int K, bool largest, float scale,
                                                                  const int *experts, const float *weights,
                                                                  const float *dweights, T *dscores, int64_t drs) {
  __shared__ float4 held[256];
  struct __attribute__((packed, aligned(sizeof(T)))) Four {
    T v[4];
  };
  const int lane = threadIdx.x & (LANES - 1);
  float4 *four = held + threadIdx.x;
  float *mine = reinterpret_cast<float *>(held + (threadIdx.x - lane));
  const float sign = largest ? scale : -scale, ninf = -__builtin_huge_valf();
  const int64_t step = (int64_t)gridDim.x * (256 / LANES);
  for (int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
    const T *s = scores + row * rs;
    T *ds = dscores + row * drs;
    int e_mine = -1;
    float w = 0.f, g = 0.f;
    if (lane < K) {
      e_mine = experts[row * K + lane];
      w = weights[row * K + lane];
      g = dweights[row * K + lane];
    }
    if (e_mine < 0) g = 0.f;
    const float inner = sum_of<LANES>(w != 0.f ? w * g : 0.f);
    const int e0 = __shfl(e_mine, 0, LANES);
    const float w0 = __shfl(w, 0, LANES);
    float top = 0.f;
    if (ALL && e0 >= 0) top = (largest ? 1.f : -1.f) * (float)s[e0];
    const float own = w != 0.f ? sign * w * (g - inner) : 0.f, rest = ALL && e0 >= 0 ? -sign * w0 * inner : 0.f;
    for (int base = 0; base < E; base += 4 * LANES) {
      const int at = base + 4 * lane, left = E - at;
      float d[4] = {};
      if (ALL && rest != 0.f && left > 0) {
        Four some;
        if (left >= 4) {
          some = *reinterpret_cast<const Four *>(s + at);
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++) some.v[i] = s[at + (i < left ? i : 0)];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float k = largest ? (float)some.v[i] : -(float)some.v[i];
          const float p = k > ninf ? other_term(k, top, scale) : 0.f;
          d[i] = p != 0.f ? rest * p : 0.f;
        }
      }
      *four = float4{d[0], d[1], d[2], d[3]};
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (e_mine >= base && e_mine < base + 4 * LANES) mine[e_mine - base] = own;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const float4 f = *four;
      const Four out{{(T)f.x, (T)f.y, (T)f.z, (T)f.w}};
      if (left >= 4) {
        *reinterpret_cast<Four *>(ds + at) = out;
      } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
          if (i < left) ds[at + i] = out.v[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// Scores and gradients of one expert side by side: a lane has a row. Its chosen experts in ascending order, so that
// one comparison an expert tells whether the next of them is reached.
template <typename T, bool ALL, int KT>
__global__ __launch_bounds__(256) void route_backward_columns_kernel(const T *scores, int64_t es, int64_t rows, int E,
                                                                     int K, bool largest, float scale,
                                                                     const int *experts, const float *weights,
                                                                     const float *dweights, T *dscores, int64_t des) {
  const float sign = largest ? scale : -scale, ninf = -__builtin_huge_valf();
  const int lo = (int)((int64_t)E * blockIdx.y / gridDim.y), hi = (int)((int64_t)E * (blockIdx.y + 1) / gridDim.y);
  for (int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x; row < rows; row += (int64_t)gridDim.x * 256) {
    int id[KT];
    float d[KT], inner = 0.f;
    float w0 = 0.f;
    int e0 = -1;
#pragma unroll
    for (int j = 0; j < KT; j++) {
      id[j] = j < K ? experts[row * K + j] : -1;
      const float w = j < K ? weights[row * K + j] : 0.f;
      const float g = id[j] >= 0 ? dweights[row * K + j] : 0.f;
      inner += w != 0.f ? w * g : 0.f;
      d[j] = g;
      if (j == 0) {
        e0 = id[0];
        w0 = w;
      }
    }
#pragma unroll
    for (int j = 0; j < KT; j++) {
      const float w = j < K ? weights[row * K + j] : 0.f;
      d[j] = w != 0.f ? sign * w * (d[j] - inner) : 0.f;
    }
    float top = 0.f;
    if (ALL && e0 >= 0) top = (largest ? 1.f : -1.f) * (float)scores[row + e0 * es];
    const float rest = ALL && e0 >= 0 ? -sign * w0 * inner : 0.f;
    // ascending experts, those that are none (and those before this stretch) last
#pragma unroll
    for (int j = 0; j < KT; j++) id[j] = id[j] >= lo ? id[j] : 0x7fffffff;
#pragma unroll
    for (int a = 0; a < KT - 1; a++)
#pragma unroll
      for (int b = 0; b < KT - 1 - a; b++) {
        const bool swap = id[b] > id[b + 1];
        const int i = swap ? id[b] : id[b + 1];
        const float v = swap ? d[b] : d[b + 1];
        id[b] = swap ? id[b + 1] : id[b];
        d[b] = swap ? d[b + 1] : d[b];
        id[b + 1] = i;
        d[b + 1] = v;
      }
    for (int u0 = lo; u0 < hi; u0 += 8) {
      T v[8];
      if (ALL) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = scores[row + (int64_t)(u0 + i < hi ? u0 + i : hi - 1) * es];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        if (u0 + i >= hi) break;
        float out = 0.f;
        if (ALL) {
          const float k = largest ? (float)v[i] : -(float)v[i];
          const float p = k > ninf ? other_term(k, top, scale) : 0.f;
          out = p != 0.f && rest != 0.f ? rest * p : 0.f;
        }
        if (u0 + i == id[0]) {
          out = d[0];
#pragma unroll
          for (int j = 0; j < KT - 1; j++) {
            id[j] = id[j + 1];
            d[j] = d[j + 1];
          }
          id[KT - 1] = 0x7fffffff;
        }
        dscores[row + (int64_t)(u0 + i) * des] = (T)out;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// order by expert: a stable counting sort
// ---------------------------------------------------------------------------

// A workgroup of up to 8 wavefronts has a chunk of slots, each wavefront a stretch of it, 64 slots at a time and at
// most SORT_STEPS times. Two slots of a wavefront find that they name the same expert by comparing a bit of
// all 64 numbers at a time, so that no order depends on when an addition happens. 16384 x 4 slots of 64 experts: 4 us
// to count and 7 to place; 100003 x 3 of 1000: 5, 5 to add up and 9 to place; 32 slots: 3, one launch.
static const int SORT_STEPS = 4, SORT_WAVES = 8;
static const size_t SORT_LDS = 150u << 10;

// How a launch cuts its slots. One workgroup: a single launch. Some: their histograms first, which every
// placing workgroup adds up by itself. More than SORT_SCAN: a third launch adds them up in between.
static const int SORT_SCAN = 64;
struct SortShape {
  int waves, chunk, blocks;
};
static SortShape sort_shape(size_t slots, int experts) {
  SortShape s;
  s.waves = SORT_WAVES;
  while (s.waves > 1 && (((size_t)s.waves * (experts + 2) + 2 * (experts + 1)) * sizeof(int) > SORT_LDS || (size_t)s.waves * 32 >= slots))
    s.waves >>= 1;
  s.chunk = s.waves * WAVE * SORT_STEPS;
  s.blocks = (int)((slots + s.chunk - 1) / s.chunk);
  if (s.blocks < 1) s.blocks = 1;
  return s;
}

__device__ __forceinline__ int bucket_of(int e, int E) { return (unsigned)e < (unsigned)E ? e : E; }

__global__ __launch_bounds__(512) void expert_count_kernel(const int *experts, int64_t slots, int E, int chunk,
                                                           int *hist) {
  extern __shared__ int cnt[];
  for (int i = threadIdx.x; i <= E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * chunk;
  const int64_t hi = lo + chunk < slots ? lo + chunk : slots;
#pragma unroll 4
  for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&cnt[bucket_of(experts[i], E)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i <= E; i += blockDim.x) hist[(int64_t)blockIdx.x * (E + 1) + i] = cnt[i];
}

// hist[c][b] -> how many of bucket b are in the chunks before c; the last row receives the totals. A wavefront
// has a bucket, its lanes chunks in a row.
__global__ __launch_bounds__(256) void expert_scan_kernel(int *hist, int blocks, int B) {
  const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  int before = 0;
  for (int c0 = 0; c0 < blocks; c0 += WAVE) {
    const int c = c0 + lane;
    const int h = c < blocks ? hist[(int64_t)c * B + b] : 0;
    int sum = h;
    for (int m = 1; m < WAVE; m <<= 1) {
      const int add = __shfl_up(sum, m, WAVE);
      if (lane >= m) sum += add;
    }
    if (c < blocks) hist[(int64_t)c * B + b] = before + sum - h;
    before += __shfl(sum, WAVE - 1, WAVE);
  }
  if (lane == 0) hist[(int64_t)blocks * B + b] = before;
}

// LDS: counters [waves][E + 1], a sum per wavefront, and where the histograms are added up here totals and
// counts before [E + 1] each. scanned: hist is expert_scan_kernel's.
__global__ __launch_bounds__(512) void expert_place_kernel(const int *experts, int64_t slots, int E, int bits, int chunk,
                                                           const int *hist, int blocks, bool scanned, int *order,
                                                           int *position, int *offsets) {
  extern __shared__ int lds[];
  const int B = E + 1, waves = blockDim.x / WAVE, lane = threadIdx.x & 63, w = threadIdx.x / WAVE;
  int *cnt = lds, *sums = lds + waves * B, *totals = sums + waves, *befores = totals + B;
  const int64_t lo = (int64_t)blockIdx.x * chunk;
  const int64_t hi = lo + chunk < slots ? lo + chunk : slots;
  const int64_t part = ((hi - lo + waves - 1) / waves + WAVE - 1) / WAVE * WAVE;
  const int64_t wlo = lo + w * part, whi = wlo + part < hi ? wlo + part : hi;
  int id[SORT_STEPS], local[SORT_STEPS];
#pragma unroll
  for (int k = 0; k < SORT_STEPS; k++) {
    const int64_t i = wlo + k * WAVE + lane;
    id[k] = i < whi ? experts[i] : 0;
  }
  const int per = (B + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * per;
  for (int i = threadIdx.x; i < waves * B; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  // place of a slot among its wavefront's of the same expert
#pragma unroll
  for (int k = 0; k < SORT_STEPS; k++) {
    if (wlo + k * WAVE >= whi) break;
    const bool in = wlo + k * WAVE + lane < whi;
    const int b = bucket_of(id[k], E);
    unsigned long long same = __ballot(in);
    for (int t = 0; t < bits; t++) {
      const bool bit = (b >> t) & 1;
      const unsigned long long v = __ballot(bit);
      same &= bit ? v : ~v;
    }
    id[k] = b;
    if (in) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int start = cnt[w * B + b];
      local[k] = start + rank;
      __builtin_amdgcn_wave_barrier();
      if (rank == 0) cnt[w * B + b] = start + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  // every bucket's place for this chunk: how many are in all, and in the chunks before
  int sum = 0;
  for (int b = b0; b < b0 + per && b < B; b++) {
    int total = 0, before = 0;
    if (blocks == 1) {
      for (int v = 0; v < waves; v++) total += cnt[v * B + b];
    } else if (scanned) {
      total = hist[(int64_t)blocks * B + b];
    } else {
#pragma unroll 16
      for (int c = 0; c < blocks; c++) {
        const int h = hist[(int64_t)c * B + b];
        total += h;
        before += c < (int)blockIdx.x ? h : 0;
      }
    }
    if (blocks > 1 && !scanned) {
      totals[b] = total;
      befores[b] = before;
    }
    sum += total;
  }
  int upto = sum;
  for (int m = 1; m < WAVE; m <<= 1) {
    const int add = __shfl_up(upto, m, WAVE);
    if (lane >= m) upto += add;
  }
  if (lane == WAVE - 1) sums[w] = upto;
  __syncthreads();
  int at = upto - sum;
  for (int v = 0; v < w; v++) at += sums[v];
  for (int b = b0; b < b0 + per && b < B; b++) {
    if (blockIdx.x == 0) offsets[b] = at;
    int run = at, next = at;
    if (scanned) {
      next += hist[(int64_t)blocks * B + b];
      run += hist[(int64_t)blockIdx.x * B + b];
    } else if (blocks > 1) {
      next += totals[b];
      run += befores[b];
    }
    for (int v = 0; v < waves; v++) {
      const int c = cnt[v * B + b];
      cnt[v * B + b] = run;
      run += c;
    }
    at = blocks > 1 ? next : run;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < SORT_STEPS; k++) {
    const int64_t i = wlo + k * WAVE + lane;
    if (i < whi) {
      const int p = cnt[w * B + id[k]] + local[k];
      order[p] = (int)i;
      position[i] = id[k] < E ? p : ~p;
    }
  }
}

// ---------------------------------------------------------------------------
// rows out and back
// ---------------------------------------------------------------------------

// Rows move in pieces of 16 bytes, at addresses that are only aligned to their elements (one load or store all
// the same); the elements behind a row's last whole piece move one by one.
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef unsigned uintx4_u __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  // ONCE: past the caches (see moves_once)
  template <bool ONCE>
  static __device__ __forceinline__ uintx4 load(const T *row, int piece) {
    const uintx4_u *at = reinterpret_cast<const uintx4_u *>(row + (int64_t)piece * N);
    return ONCE ? __builtin_nontemporal_load(at) : *at;
  }
  template <bool ONCE>
  static __device__ __forceinline__ void store(T *row, int piece, uintx4 v) {
    uintx4_u *at = reinterpret_cast<uintx4_u *>(row + (int64_t)piece * N);
    if (ONCE)
      __builtin_nontemporal_store((uintx4_u)v, at);
    else
      *at = v;
  }
  static __device__ __forceinline__ void unpack(uintx4 v, float (&f)[N]) {
    T e[N];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = (float)e[i];
  }
  static __device__ __forceinline__ uintx4 pack(const float (&f)[N]) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; i++) e[i] = (T)f[i];
    uintx4 v;
    __builtin_memcpy(&v, e, 16);
    return v;
  }
};

// How the threads of a launch share the tokens' rows: 2^lanes_log2 lanes to a row (as many as it has pieces, 64
// at most), U pieces each, and blockIdx.y further stretches of a long row. Neighbouring lanes have
// neighbouring pieces.
struct RowShare {
  int64_t tokens;
  int K, d, lanes_log2;
};

// dst[place(t, j)] = src[t], zeros where the slot has no expert. A row is read once for its top_k places. Memory
// bounds it: 16384 x 2048 bfloat16, four places, 54 us, 6.2 TB/s, mostly writes.
template <typename T, int U, bool ONCE>
__global__ __launch_bounds__(256) void send_rows_kernel(const T *src, int64_t ss, const int *position, RowShare a,
                                                        T *dst, int64_t ds) {
  constexpr int N = Row<T>::N;
  const int lanes = 1 << a.lanes_log2, whole = a.d / N, lane = threadIdx.x & (lanes - 1);
  const int first = (int)blockIdx.y * lanes * U + lane;
  const int64_t step = (int64_t)gridDim.x * (256 >> a.lanes_log2);
  for (int64_t t = (int64_t)blockIdx.x * (256 >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2); t < a.tokens; t += step) {
    const T *row = src + t * ss;
    uintx4 p[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (first + u * lanes < whole) p[u] = Row<T>::template load<ONCE>(row, first + u * lanes);
    for (int j = 0; j < a.K; j++) {
      const int at = position[t * a.K + j];
      T *to = dst + (int64_t)(at < 0 ? ~at : at) * ds;
#pragma unroll
      for (int u = 0; u < U; u++)
        if (first + u * lanes < whole) Row<T>::template store<false>(to, first + u * lanes, at < 0 ? uintx4{0, 0, 0, 0} : p[u]);
    }
    if (blockIdx.y == 0)
      for (int c = whole * N + lane; c < a.d; c += lanes) {
        const T v = row[c];
        for (int j = 0; j < a.K; j++) {
          const int at = position[t * a.K + j];
          dst[(int64_t)(at < 0 ? ~at : at) * ds + c] = at < 0 ? (T)0.f : v;
        }
      }
  }
}

// dst[t] = sum over j of (w[t][j] *) src[place(t, j)], j ascending; four rows of them on their way at a time.
// Memory bounds it: 16384 x 2048 bfloat16, four places, 57 us, 5.9 TB/s.
template <typename T, int U, bool WEIGHTED, bool ONCE, bool PUT_ONCE>
__global__ __launch_bounds__(256) void join_rows_kernel(const T *src, int64_t ss, const float *w, const int *position,
                                                        RowShare a, T *dst, int64_t ds) {
  constexpr int N = Row<T>::N;
  const int lanes = 1 << a.lanes_log2, whole = a.d / N, lane = threadIdx.x & (lanes - 1);
  const int first = (int)blockIdx.y * lanes * U + lane, stride = gridDim.y * lanes * U;
  const int64_t step = (int64_t)gridDim.x * (256 >> a.lanes_log2);
  for (int64_t t = (int64_t)blockIdx.x * (256 >> a.lanes_log2) + (threadIdx.x >> a.lanes_log2); t < a.tokens; t += step) {
    for (int i0 = first; i0 < whole; i0 += stride) {
      float acc[U][N] = {};
      for (int j0 = 0; j0 < a.K; j0 += 4) {
        int at[4];
        float by[4];
        uintx4 p[4][U];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          at[j] = j0 + j < a.K ? position[t * a.K + j0 + j] : -1;
          by[j] = WEIGHTED && j0 + j < a.K ? w[t * a.K + j0 + j] : 1.f;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
          for (int u = 0; u < U; u++)
            if (at[j] >= 0 && i0 + u * lanes < whole)
              p[j][u] = Row<T>::template load<ONCE>(src + (int64_t)at[j] * ss, i0 + u * lanes);
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (at[j] >= 0) {
#pragma unroll
            for (int u = 0; u < U; u++) {
              float v[N];
              Row<T>::unpack(p[j][u], v);
#pragma unroll
              for (int e = 0; e < N; e++) acc[u][e] = WEIGHTED ? fmaf(by[j], v[e], acc[u][e]) : acc[u][e] + v[e];
            }
          }
      }
#pragma unroll
      for (int u = 0; u < U; u++)
        if (i0 + u * lanes < whole) Row<T>::template store<PUT_ONCE>(dst + t * ds, i0 + u * lanes, Row<T>::pack(acc[u]));
    }
    if (blockIdx.y == 0)
      for (int c = whole * N + lane; c < a.d; c += lanes) {
        float sum = 0.f;
        for (int j = 0; j < a.K; j++) {
          const int at = position[t * a.K + j];
          if (at < 0) continue;
          const float v = (float)src[(int64_t)at * ss + c];
          sum = WEIGHTED ? fmaf(w[t * a.K + j], v, sum) : sum + v;
        }
        dst[t * ds + c] = (T)sum;
      }
  }
}

// Both gradients of the weighted sum in one pass over the rows: J of a token's places at a time. SPLIT: the
// four wavefronts of a workgroup share a token's row, otherwise each has tokens of its own. 16384 x 2048 bfloat16,
// four places: 94 us, 6.4 TB/s.
template <typename T, int U, int J, bool SPLIT, bool ONCE>
__global__ __launch_bounds__(256) void join_backward_kernel(const T *dout, int64_t os, const T *rows, int64_t rs,
                                                            const float *w, const int *position, RowShare a,
                                                            T *drows, int64_t drs, float *dw) {
  constexpr int N = Row<T>::N;
  __shared__ float part[SPLIT ? 4 * J : 1];
  const int lanes = 1 << a.lanes_log2, whole = a.d / N, wave = threadIdx.x >> 6;
  const int lane = SPLIT ? threadIdx.x : threadIdx.x & (lanes - 1), stride = SPLIT ? 256 : lanes;
  const int per = SPLIT ? 1 : 256 >> a.lanes_log2, width = SPLIT ? WAVE : lanes;
  const int64_t step = (int64_t)gridDim.x * per;
  for (int64_t t = (int64_t)blockIdx.x * per + (SPLIT ? 0 : threadIdx.x >> a.lanes_log2); t < a.tokens; t += step) {
    const T *g_row = dout + t * os;
    for (int j0 = 0; j0 < a.K; j0 += J) {
      int at[J];
      float by[J], dot[J] = {};
#pragma unroll
      for (int j = 0; j < J; j++) {
        at[j] = j0 + j < a.K ? position[t * a.K + j0 + j] : -1;
        by[j] = j0 + j < a.K ? w[t * a.K + j0 + j] : 0.f;
      }
      for (int i0 = lane; i0 < whole; i0 += stride * U) {
        uintx4 g[U], y[J][U];
#pragma unroll
        for (int u = 0; u < U; u++)
          if (i0 + u * stride < whole) g[u] = Row<T>::template load<ONCE>(g_row, i0 + u * stride);
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
          for (int u = 0; u < U; u++)
            if (at[j] >= 0 && i0 + u * stride < whole) y[j][u] = Row<T>::template load<ONCE>(rows + (int64_t)at[j] * rs, i0 + u * stride);
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (i0 + u * stride >= whole) break;
          float gv[N];
          Row<T>::unpack(g[u], gv);
#pragma unroll
          for (int j = 0; j < J; j++) {
            if (at[j] >= 0) {
              float yv[N], out[N];
              Row<T>::unpack(y[j][u], yv);
#pragma unroll
              for (int e = 0; e < N; e++) {
                dot[j] = fmaf(gv[e], yv[e], dot[j]);
                out[e] = by[j] * gv[e];
              }
              Row<T>::template store<false>(drows + (int64_t)at[j] * drs, i0 + u * stride, Row<T>::pack(out));
            } else if (j0 + j < a.K) {
              Row<T>::template store<false>(drows + (int64_t)~at[j] * drs, i0 + u * stride, uintx4{0, 0, 0, 0});
            }
          }
        }
      }
      for (int c = whole * N + lane; c < a.d; c += stride) {
        const float gv = (float)g_row[c];
#pragma unroll
        for (int j = 0; j < J; j++) {
          if (j0 + j >= a.K) break;
          if (at[j] >= 0) dot[j] = fmaf(gv, (float)rows[(int64_t)at[j] * rs + c], dot[j]);
          drows[(int64_t)(at[j] < 0 ? ~at[j] : at[j]) * drs + c] = at[j] < 0 ? (T)0.f : (T)(by[j] * gv);
        }
      }
#pragma unroll
      for (int j = 0; j < J; j++)
        for (int m = width >> 1; m >= 1; m >>= 1) dot[j] += __shfl_xor(dot[j], m, WAVE);
      if (SPLIT) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
          for (int j = 0; j < J; j++) part[wave * J + j] = dot[j];
        }
        __syncthreads();
        if (threadIdx.x < J && j0 + (int)threadIdx.x < a.K)
          dw[t * a.K + j0 + threadIdx.x] = (part[threadIdx.x] + part[J + threadIdx.x]) +
                                           (part[2 * J + threadIdx.x] + part[3 * J + threadIdx.x]);
      } else if (lane == 0) {
#pragma unroll
        for (int j = 0; j < J; j++)
          if (j0 + j < a.K) dw[t * a.K + j0 + j] = dot[j];
      }
    }
  }
}

// Whether rows are read (and a joined row is written) past the caches: with more than the L2s hold they are not read
// again before they have left them, and keeping them costs (16384 x 2048 bfloat16, four places: joined 57 us against
// 94, sent 55 against 58, both gradients 106 against 111). Rows that are no whole cache lines share some with their
// neighbours and are read better through the caches (100003 x 101 float: 46 us against 49, sent 45 against 53;
// 200000 x 32 float16, eight places, both gradients: 63 us against 85).
static bool moves_once(size_t rows, size_t cols, size_t elem) { return rows * cols * elem > (size_t)(32 << 20); }
static bool whole_lines(const void *p, size_t stride, size_t elem) {
  return aligned_to(p, 128) && stride * elem % 128 == 0;
}

// The share of rows of d elements of T, U pieces to a lane, and its grid.
template <typename T>
static RowShare share_rows(size_t tokens, int top_k, size_t cols, int U, dim3 *grid) {
  RowShare a;
  a.tokens = (int64_t)tokens;
  a.K = top_k;
  a.d = (int)cols;
  const int pieces = (int)((cols + Row<T>::N - 1) / Row<T>::N);
  a.lanes_log2 = 0;
  while (a.lanes_log2 < 6 && (1 << a.lanes_log2) * U < pieces) a.lanes_log2++;
  const int lanes = 1 << a.lanes_log2;
  const size_t per = 256 >> a.lanes_log2;
  *grid = dim3(grid_of((tokens + per - 1) / per), (unsigned)((pieces + lanes * U - 1) / (lanes * U)));
  return a;
}

// ---------------------------------------------------------------------------
// checks
// ---------------------------------------------------------------------------

static const size_t MOST_ROWS = 2147483646;   // places are int32, and ~place is one too
static const size_t MOST_COLS = 1000000;

static bool choice_ok(size_t rows, int top_k) {
  return top_k >= 1 && top_k <= H2O4GPU_EXPERTS_MAX_TOP_K && rows <= MOST_ROWS / (size_t)top_k;
}

static bool experts_ok(int experts) { return experts >= 1 && experts <= H2O4GPU_EXPERTS_MAX_EXPERTS; }

static bool rows_ok(int dtype, const void *p, size_t stride, size_t cols) {
  return p && aligned_to(p, type_size(dtype)) && stride <= ((size_t)1 << 40) && (stride >= cols || stride == 0);
}

static bool ints_ok(const void *p) { return p && aligned_to(p, 4); }

static bool stride_ok(ptrdiff_t s) { return s <= ((ptrdiff_t)1 << 40) && s >= -((ptrdiff_t)1 << 40); }

}  // namespace kmhip

using namespace kmhip;

KM_API int h2o4gpu_experts_route(int dtype, size_t rows, int experts, int top_k, int largest, int over_all,
                                 float scale, const void *d_scores, ptrdiff_t row_stride, ptrdiff_t expert_stride,
                                 int *d_experts, float *d_weights, void *stream) {
  if (!known_type(dtype) || !experts_ok(experts) || !choice_ok(rows, top_k) || top_k > experts ||
      !(scale >= 0.f) || !isfinite(scale) || !stride_ok(row_stride) || !stride_ok(expert_stride))
    return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!d_scores || !aligned_to(d_scores, type_size(dtype)) || !ints_ok(d_experts) || !ints_ok(d_weights))
    return H2O4GPU_KMEANS_EARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    const T *scores = static_cast<const T *>(d_scores);
    const int64_t n = (int64_t)rows;
    // columns: lists of up to eight stay in registers (longer ones go the general way)
    if (row_stride == 1 && expert_stride != 1 && top_k <= 8) {
      const auto columns = [&](auto all, auto kt) {
        constexpr int KT = decltype(kt)::value;
        int parts = 1;  // until there are some 2048 wavefronts, or a stretch is as short as a load's eight
        while (parts < 16 && (n + 63) / 64 * parts < 2048 && experts / (parts * 2) >= 8) parts *= 2;
        auto kernel = route_columns_kernel<T, decltype(all)::value, KT>;
        const size_t lds = parts > 1 ? sizeof(float) * parts * (2 * KT + 1) * 64 : 0;  // (68 KB for 16 lists of eight)
        KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(kernel), lds));
        hipLaunchKernelGGL(kernel, dim3(grid_of((rows + 63) / 64)), dim3(64 * parts), lds, s, scores,
                           (int64_t)expert_stride, n, experts, top_k, largest != 0, scale, d_experts, d_weights);
        return launched();
      };
      const auto by_k = [&](auto all) {
        return top_k == 1 ? columns(all, Int<1>()) : top_k == 2 ? columns(all, Int<2>())
               : top_k <= 4 ? columns(all, Int<4>()) : columns(all, Int<8>());
      };
      return over_all ? by_k(Int<1>()) : by_k(Int<0>());
    }
    const auto in_rows = [&](auto lanes, auto nv) {
      constexpr int L = decltype(lanes)::value, NV = decltype(nv)::value;
      auto kernel = over_all ? route_rows_kernel<T, true, L, NV> : route_rows_kernel<T, false, L, NV>;
      hipLaunchKernelGGL(kernel, dim3(grid_of((rows * L + 255) / 256)), dim3(256), 0, s, scores, (int64_t)row_stride, n,
                         experts, top_k, largest != 0, scale, d_experts, d_weights);
      return launched();
    };
    if (expert_stride == 1 && experts <= 1024) {
      if (experts <= 16 && top_k <= 4) return in_rows(Int<4>(), Int<4>());
      if (experts <= 64 && top_k <= 16) return in_rows(Int<16>(), Int<4>());
      if (experts <= 256 && top_k <= 16) return in_rows(Int<16>(), Int<16>());
      return in_rows(Int<64>(), Int<16>());
    }
    auto kernel = largest ? (over_all ? route_any_kernel<T, true, true> : route_any_kernel<T, true, false>)
                          : (over_all ? route_any_kernel<T, false, true> : route_any_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3(grid_of((rows + 3) / 4)), dim3(256), 0, s, scores, (int64_t)row_stride,
                       (int64_t)expert_stride, n, experts, top_k, scale, d_experts, d_weights);
    return launched();
  });
}

KM_API int h2o4gpu_experts_route_backward(int dtype, size_t rows, int experts, int top_k, int largest, int over_all,
                                          float scale, const void *d_scores, ptrdiff_t row_stride,
                                          ptrdiff_t expert_stride, const int *d_experts, const float *d_weights,
                                          const float *d_dweights, void *d_dscores, ptrdiff_t drow_stride,
                                          ptrdiff_t dexpert_stride, void *stream) {
  if (!known_type(dtype) || !experts_ok(experts) || !choice_ok(rows, top_k) || top_k > experts ||
      !(scale >= 0.f) || !isfinite(scale) || !stride_ok(row_stride) || !stride_ok(expert_stride) ||
      !stride_ok(drow_stride) || !stride_ok(dexpert_stride))
    return H2O4GPU_KMEANS_EARG;
  if (rows == 0) return H2O4GPU_KMEANS_OK;
  if (!d_scores || !aligned_to(d_scores, type_size(dtype)) || !d_dscores ||
      !aligned_to(d_dscores, type_size(dtype)) || !ints_ok(d_experts) || !ints_ok(d_weights) || !ints_ok(d_dweights))
    return H2O4GPU_KMEANS_EARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    const T *scores = static_cast<const T *>(d_scores);
    T *dscores = static_cast<T *>(d_dscores);
    const int64_t n = (int64_t)rows;
    if (row_stride == 1 && drow_stride == 1 && dexpert_stride != 1 && top_k <= 8) {
      unsigned parts = 1;
      while ((n + 255) / 256 * parts < 512 && experts / (int)(parts * 2) >= 16) parts *= 2;
      const dim3 grid(grid_of((rows + 255) / 256), parts);
      const auto columns = [&](auto kt) {
        constexpr int KT = decltype(kt)::value;
        auto kernel = over_all ? route_backward_columns_kernel<T, true, KT> : route_backward_columns_kernel<T, false, KT>;
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, scores, (int64_t)expert_stride, n, experts, top_k, largest != 0,
                           scale, d_experts, d_weights, d_dweights, dscores, (int64_t)dexpert_stride);
        return launched();
      };
      return top_k <= 2 ? columns(Int<2>()) : top_k <= 4 ? columns(Int<4>()) : columns(Int<8>());
    }
    if (expert_stride == 1 && dexpert_stride == 1) {
      const auto in_rows = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        auto kernel = over_all ? route_backward_rows_kernel<T, true, L> : route_backward_rows_kernel<T, false, L>;
        hipLaunchKernelGGL(kernel, dim3(grid_of((rows * L + 255) / 256)), dim3(256), 0, s, scores, (int64_t)row_stride, n,
                           experts, top_k, largest != 0, scale, d_experts, d_weights, d_dweights, dscores,
                           (int64_t)drow_stride);
        return launched();
      };
      return experts <= 16 && top_k <= 4    ? in_rows(Int<4>())
             : experts <= 64 && top_k <= 16 ? in_rows(Int<16>())
                                            : in_rows(Int<64>());
    }
    auto kernel = over_all ? route_backward_kernel<T, true> : route_backward_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3(grid_of((rows + 3) / 4)), dim3(256), 0, s, scores, (int64_t)row_stride,
                       (int64_t)expert_stride, n, experts, top_k, largest != 0, scale, d_experts, d_weights, d_dweights,
                       dscores, (int64_t)drow_stride, (int64_t)dexpert_stride);
    return launched();
  });
}

KM_API size_t h2o4gpu_experts_sort_workspace(size_t slots, int experts) {
  if (!experts_ok(experts) || slots > MOST_ROWS) return 0;
  const int blocks = sort_shape(slots, experts).blocks;
  return blocks > 1 ? (size_t)(blocks + 1) * (experts + 1) * sizeof(int) : 0;
}

KM_API int h2o4gpu_experts_sort(size_t slots, int experts, const int *d_experts, int *d_order, int *d_position,
                                int *d_offsets, void *d_workspace, size_t workspace_bytes, void *stream) {
  if (!experts_ok(experts) || slots > MOST_ROWS || !ints_ok(d_offsets)) return H2O4GPU_KMEANS_EARG;
  if (slots > 0 && (!ints_ok(d_experts) || !ints_ok(d_order) || !ints_ok(d_position))) return H2O4GPU_KMEANS_EARG;
  const size_t need = h2o4gpu_experts_sort_workspace(slots, experts);
  if (need > 0 && (!ints_ok(d_workspace) || workspace_bytes < need)) return H2O4GPU_KMEANS_EARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int buckets = experts + 1;
  const SortShape shape = sort_shape(slots, experts);
  int *hist = static_cast<int *>(d_workspace);
  // (with very many buckets there is no room for what is added up)
  const bool scanned = shape.blocks > SORT_SCAN || (shape.blocks > 1 && shape.waves == 1);
  int bits = 0;
  while ((experts >> bits) != 0) bits++;
  if (shape.blocks > 1) {
    const size_t lds = (size_t)buckets * sizeof(int);
    KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(expert_count_kernel), lds));
    hipLaunchKernelGGL(expert_count_kernel, dim3(shape.blocks), dim3(512), lds, s, d_experts, (int64_t)slots, experts,
                       shape.chunk, hist);
    KM_TRY(launched());
    if (scanned) {
      hipLaunchKernelGGL(expert_scan_kernel, dim3((buckets + 3) / 4), dim3(256), 0, s, hist, shape.blocks, buckets);
      KM_TRY(launched());
    }
  }
  const size_t lds = ((size_t)shape.waves * (buckets + 1) + (shape.blocks > 1 && !scanned ? 2 * buckets : 0)) * sizeof(int);
  KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(expert_place_kernel), lds));
  hipLaunchKernelGGL(expert_place_kernel, dim3(shape.blocks), dim3(shape.waves * WAVE), lds, s, d_experts,
                     (int64_t)slots, experts, bits, shape.chunk, hist, shape.blocks, scanned, d_order, d_position,
                     d_offsets);
  return launched();
}

KM_API int h2o4gpu_experts_dispatch(int dtype, size_t tokens, int top_k, size_t cols, const void *d_x,
                                    size_t x_stride, const int *d_position, void *d_rows, size_t rows_stride,
                                    void *stream) {
  if (!known_type(dtype) || !choice_ok(tokens, top_k) || cols < 1 || cols > MOST_COLS) return H2O4GPU_KMEANS_EARG;
  if (tokens == 0) return H2O4GPU_KMEANS_OK;
  if (!rows_ok(dtype, d_x, x_stride, cols) || !rows_ok(dtype, d_rows, rows_stride, cols) || rows_stride < cols ||
      !ints_ok(d_position))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    dim3 grid;
    const RowShare a = share_rows<T>(tokens, top_k, cols, 4, &grid);
    const bool once = moves_once(tokens * top_k, cols, sizeof(T)) && whole_lines(d_x, x_stride, sizeof(T));
    hipLaunchKernelGGL((once ? send_rows_kernel<T, 4, true> : send_rows_kernel<T, 4, false>), grid, dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<const T *>(d_x), (int64_t)x_stride, d_position, a,
                       static_cast<T *>(d_rows), (int64_t)rows_stride);
    return launched();
  });
}

static int join_rows(int dtype, size_t tokens, int top_k, size_t cols, const void *src, size_t src_stride,
                     const float *w, bool weighted, const int *position, void *dst, size_t dst_stride,
                     void *stream) {
  if (!known_type(dtype) || !choice_ok(tokens, top_k) || cols < 1 || cols > MOST_COLS) return H2O4GPU_KMEANS_EARG;
  if (tokens == 0) return H2O4GPU_KMEANS_OK;
  if (!rows_ok(dtype, src, src_stride, cols) || !rows_ok(dtype, dst, dst_stride, cols) || dst_stride < cols ||
      !ints_ok(position) || (weighted && !ints_ok(w)))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    dim3 grid;
    // short rows: a piece a lane (60000 x 515 bfloat16, three places: 61 us against 71 with two); long ones: four
    // (16384 x 2048, four places: 81 against 85)
    const bool short_rows = cols <= 128 * Row<T>::N;
    const RowShare a = share_rows<T>(tokens, top_k, cols, short_rows ? 1 : 4, &grid);
    if (tokens >= 4096) grid.y = 1;  // (enough rows for every wavefront to have whole ones)
    const bool put_once = moves_once(tokens * top_k, cols, sizeof(T));
    const bool once = put_once && whole_lines(src, src_stride, sizeof(T));
    const auto pick = [&](auto u, auto by_weight) {
      constexpr int U = decltype(u)::value;
      constexpr bool W = decltype(by_weight)::value != 0;
      return once       ? join_rows_kernel<T, U, W, true, true>
             : put_once ? join_rows_kernel<T, U, W, false, true>
                        : join_rows_kernel<T, U, W, false, false>;
    };
    auto kernel = short_rows ? (weighted ? pick(Int<1>(), Int<1>()) : pick(Int<1>(), Int<0>()))
                             : (weighted ? pick(Int<4>(), Int<1>()) : pick(Int<4>(), Int<0>()));
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const T *>(src),
                       (int64_t)src_stride, w, position, a, static_cast<T *>(dst), (int64_t)dst_stride);
    return launched();
  });
}

KM_API int h2o4gpu_experts_dispatch_backward(int dtype, size_t tokens, int top_k, size_t cols, const void *d_drows,
                                             size_t rows_stride, const int *d_position, void *d_dx, size_t x_stride,
                                             void *stream) {
  return join_rows(dtype, tokens, top_k, cols, d_drows, rows_stride, nullptr, false, d_position, d_dx, x_stride,
                   stream);
}

KM_API int h2o4gpu_experts_combine(int dtype, size_t tokens, int top_k, size_t cols, const void *d_rows,
                                   size_t rows_stride, const float *d_weights, const int *d_position, void *d_out,
                                   size_t out_stride, void *stream) {
  return join_rows(dtype, tokens, top_k, cols, d_rows, rows_stride, d_weights, true, d_position, d_out, out_stride,
                   stream);
}

KM_API int h2o4gpu_experts_combine_backward(int dtype, size_t tokens, int top_k, size_t cols, const void *d_dout,
                                            size_t dout_stride, const void *d_rows, size_t rows_stride,
                                            const float *d_weights, const int *d_position, void *d_drows,
                                            size_t drows_stride, float *d_dweights, void *stream) {
  if (!known_type(dtype) || !choice_ok(tokens, top_k) || cols < 1 || cols > MOST_COLS) return H2O4GPU_KMEANS_EARG;
  if (tokens == 0) return H2O4GPU_KMEANS_OK;
  if (!rows_ok(dtype, d_dout, dout_stride, cols) || !rows_ok(dtype, d_rows, rows_stride, cols) ||
      !rows_ok(dtype, d_drows, drows_stride, cols) || drows_stride < cols || !ints_ok(d_weights) ||
      !ints_ok(d_position) || !ints_ok(d_dweights))
    return H2O4GPU_KMEANS_EARG;
  return with_type(dtype, [&](auto tag) {
    typedef typename decltype(tag)::type T;
    dim3 grid;
    const RowShare a = share_rows<T>(tokens, top_k, cols, 2, &grid);
    const bool split = tokens < 1024 && grid.y > 1;  // few long rows
    const bool once = moves_once(tokens * top_k, cols, sizeof(T)) && whole_lines(d_rows, rows_stride, sizeof(T)) &&
                      whole_lines(d_dout, dout_stride, sizeof(T));
    const auto pick = [&](auto j) {
      constexpr int J = decltype(j)::value;
      return split ? join_backward_kernel<T, 2, J, true, false>
             : once ? join_backward_kernel<T, 2, J, false, true>
                    : join_backward_kernel<T, 2, J, false, false>;
    };
    auto kernel = top_k <= 2 ? pick(Int<2>()) : pick(Int<4>());
    hipLaunchKernelGGL(kernel, dim3(split ? (unsigned)tokens : grid.x), dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<const T *>(d_dout), (int64_t)dout_stride,
                       static_cast<const T *>(d_rows), (int64_t)rows_stride, d_weights, d_position, a,
                       static_cast<T *>(d_drows), (int64_t)drows_stride, d_dweights);
    return launched();
  });
}
