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

// One wavefront a row: inner = sum of w g over the chosen, then every expert's gradient.
template <typename T, bool LARGEST, bool ALL>
__global__ __launch_bounds__(256) void route_backward_kernel(const T *scores, int64_t rs, int64_t es, int64_t rows,
                                                             int E, int K, float scale, const int *experts,
                                                             const float *weights, const float *dweights,
                                                             T *dscores, int64_t drs, int64_t des) {
  const int lane = threadIdx.x & 63;
  const float sign = LARGEST ? scale : -scale;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
  int e_mine = -1;
  float w = 0.f, g = 0.f;
  if (lane < K) {
    e_mine = experts[row * K + lane];
    w = weights[row * K + lane];
    g = e_mine >= 0 ? dweights[row * K + lane] : 0.f;
  }
  float inner = e_mine >= 0 ? w * g : 0.f;
  for (int m = 32; m >= 1; m >>= 1) inner += __shfl_xor(inner, m, WAVE);
  const int e0 = __shfl(e_mine, 0, WAVE);
  const float w0 = __shfl(w, 0, WAVE);
  const float ninf = -__builtin_huge_valf();
  float top = ninf;
  if (ALL && e0 >= 0) top = score_key<LARGEST>((float)scores[row * rs + e0 * es]);
  for (int base = 0; base < E; base += WAVE) {
    const int e = base + lane;
    float p = 0.f, ge = 0.f;
    bool chosen = false;
    for (int j = 0; j < K; j++) {
      const int ej = __shfl(e_mine, j, WAVE);
      const float wj = __shfl(w, j, WAVE), gj = __shfl(g, j, WAVE);
      if (ej == e && ej >= 0) {
        p = wj;
        ge = gj;
        chosen = true;
      }
    }
    if (e >= E) continue;
    if (ALL && !chosen && e0 >= 0) {
      const float k = score_key<LARGEST>((float)scores[row * rs + e * es]);
      if (k != ninf) p = w0 * softmax_term(k, top, scale);
    }
    const float d = p != 0.f ? sign * p * (ge - inner) : 0.f;
    dscores[row * drs + e * des] = (T)d;
  }
  }
}

// ---------------------------------------------------------------------------
// order by expert: a stable counting sort
// ---------------------------------------------------------------------------

// Slots of one workgroup of the counting pass and of the placing one.
static const int SORT_CHUNK = 8192;

static int sort_blocks(size_t slots) { return (int)((slots + SORT_CHUNK - 1) / SORT_CHUNK); }

__device__ __forceinline__ int bucket_of(int e, int E) { return (unsigned)e < (unsigned)E ? e : E; }

__global__ __launch_bounds__(1024) void expert_count_kernel(const int *experts, int64_t slots, int E, int *hist) {
  extern __shared__ int cnt[];
  for (int i = threadIdx.x; i <= E; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * SORT_CHUNK;
  const int64_t hi = lo + SORT_CHUNK < slots ? lo + SORT_CHUNK : slots;
  for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&cnt[bucket_of(experts[i], E)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i <= E; i += blockDim.x) hist[(int64_t)blockIdx.x * (E + 1) + i] = cnt[i];
}

// One workgroup of `waves` wavefronts places a chunk: wavefront w has the w-th part of it and
// counters of its own, so that equal experts keep their slots' order. LDS: counters [waves][E + 1],
// scan [blockDim].
__global__ __launch_bounds__(1024) void expert_place_kernel(const int *experts, int64_t slots, int E, int bits,
                                                            const int *hist, int blocks, int *order, int *position,
                                                            int *offsets) {
  extern __shared__ int lds[];
  const int B = E + 1, waves = blockDim.x / WAVE, lane = threadIdx.x & 63, w = threadIdx.x / WAVE;
  int *cnt = lds;
  int *scan = lds + waves * B;
  for (int i = threadIdx.x; i < waves * B; i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int64_t lo = (int64_t)blockIdx.x * SORT_CHUNK;
  const int64_t hi = lo + SORT_CHUNK < slots ? lo + SORT_CHUNK : slots;
  const int64_t part = ((hi - lo + waves - 1) / waves + WAVE - 1) / WAVE * WAVE;
  const int64_t wlo = lo + w * part, whi = wlo + part < hi ? wlo + part : hi;
  for (int64_t i = wlo + lane; i < whi; i += WAVE) atomicAdd(&cnt[w * B + bucket_of(experts[i], E)], 1);
  __syncthreads();
  // every bucket's place for this chunk: thread t has `per` buckets in a row
  const int per = (B + blockDim.x - 1) / blockDim.x;
  const int b0 = threadIdx.x * per;
  int sum = 0;
  for (int b = b0; b < b0 + per && b < B; b++) {
    if (blocks == 1) {
      for (int v = 0; v < waves; v++) sum += cnt[v * B + b];
    } else {
      for (int c = 0; c < blocks; c++) sum += hist[(int64_t)c * B + b];
    }
  }
  scan[threadIdx.x] = sum;
  __syncthreads();
  for (int m = 1; m < (int)blockDim.x; m <<= 1) {
    const int add = (int)threadIdx.x >= m ? scan[threadIdx.x - m] : 0;
    __syncthreads();
    scan[threadIdx.x] += add;
    __syncthreads();
  }
  int at = scan[threadIdx.x] - sum;
  for (int b = b0; b < b0 + per && b < B; b++) {
    if (blockIdx.x == 0) offsets[b] = at;
    int total = 0, before = 0;
    if (blocks > 1) {
      for (int c = 0; c < blocks; c++) {
        const int h = hist[(int64_t)c * B + b];
        total += h;
        if (c < (int)blockIdx.x) before += h;
      }
    }
    int run = at + before;
    for (int v = 0; v < waves; v++) {
      const int c = cnt[v * B + b];
      cnt[v * B + b] = run;
      run += c;
      if (blocks == 1) total += c;
    }
    at += total;
  }
  __syncthreads();
  for (int64_t base = wlo; base < whi; base += WAVE) {
    const int64_t i = base + lane;
    const bool in = i < whi;
    const int b = in ? bucket_of(experts[i], E) : 0;
    unsigned long long same = __ballot(in);
    for (int t = 0; t < bits; t++) {
      const bool bit = (b >> t) & 1;
      const unsigned long long v = __ballot(in && bit);
      same &= bit ? v : ~v;
    }
    if (in) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int start = cnt[w * B + b];
      const int p = start + rank;
      order[p] = (int)i;
      position[i] = b < E ? p : ~p;
      __builtin_amdgcn_wave_barrier();
      if (rank == 0) cnt[w * B + b] = start + __popcll(same);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------
// rows out and back
// ---------------------------------------------------------------------------

// dst[place(t, j)] = src[t], zeros where the slot has no expert.
template <typename T>
__global__ __launch_bounds__(256) void send_rows_kernel(const T *src, int64_t ss, const int *position, int64_t tokens,
                                                        int K, int d, T *dst, int64_t ds) {
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
  for (int j = 0; j < K; j++) {
    const int p = position[t * K + j];
    T *to = dst + (int64_t)(p < 0 ? ~p : p) * ds;
    for (int c = threadIdx.x; c < d; c += blockDim.x) to[c] = p < 0 ? (T)0.f : src[t * ss + c];
  }
}

// dst[t] = sum over j of (w[t][j] *) src[place(t, j)].
template <typename T, bool WEIGHTED>
__global__ __launch_bounds__(256) void join_rows_kernel(const T *src, int64_t ss, const float *w, const int *position,
                                                        int64_t tokens, int K, int d, T *dst, int64_t ds) {
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
  for (int c = threadIdx.x; c < d; c += blockDim.x) {
    float acc = 0.f;
    for (int j = 0; j < K; j++) {
      const int p = position[t * K + j];
      if (p < 0) continue;
      const float v = (float)src[(int64_t)p * ss + c];
      acc = WEIGHTED ? fmaf(w[t * K + j], v, acc) : acc + v;
    }
    dst[t * ds + c] = (T)acc;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void join_backward_kernel(const T *dout, int64_t os, const T *rows, int64_t rs,
                                                            const float *w, const int *position, int64_t tokens,
                                                            int K, int d, T *drows, int64_t drs, float *dw) {
  __shared__ float part[4];
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x)
  for (int j = 0; j < K; j++) {
    const int p = position[t * K + j];
    const int64_t at = p < 0 ? ~p : p;
    const float wj = p < 0 ? 0.f : w[t * K + j];
    float acc = 0.f;
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      if (p < 0) {
        drows[at * drs + c] = (T)0.f;
        continue;
      }
      const float g = (float)dout[t * os + c];
      acc = fmaf(g, (float)rows[at * rs + c], acc);
      drows[at * drs + c] = (T)(wj * g);
    }
    for (int m = 32; m >= 1; m >>= 1) acc += __shfl_xor(acc, m, WAVE);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) dw[t * K + j] = (part[0] + part[1]) + (part[2] + part[3]);
  }
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
    auto kernel = largest ? (over_all ? route_any_kernel<T, true, true> : route_any_kernel<T, true, false>)
                          : (over_all ? route_any_kernel<T, false, true> : route_any_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3(grid_of((rows + 3) / 4)), dim3(256), 0, s, static_cast<const T *>(d_scores),
                       (int64_t)row_stride, (int64_t)expert_stride, (int64_t)rows, experts, top_k, scale, d_experts,
                       d_weights);
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
    auto kernel = largest ? (over_all ? route_backward_kernel<T, true, true> : route_backward_kernel<T, true, false>)
                          : (over_all ? route_backward_kernel<T, false, true>
                                      : route_backward_kernel<T, false, false>);
    hipLaunchKernelGGL(kernel, dim3(grid_of((rows + 3) / 4)), dim3(256), 0, s, static_cast<const T *>(d_scores),
                       (int64_t)row_stride, (int64_t)expert_stride, (int64_t)rows, experts, top_k, scale, d_experts,
                       d_weights, d_dweights, static_cast<T *>(d_dscores), (int64_t)drow_stride,
                       (int64_t)dexpert_stride);
    return launched();
  });
}

KM_API size_t h2o4gpu_experts_sort_workspace(size_t slots, int experts) {
  if (!experts_ok(experts) || slots > MOST_ROWS) return 0;
  const int blocks = sort_blocks(slots);
  return blocks > 1 ? (size_t)blocks * (experts + 1) * sizeof(int) : 0;
}

KM_API int h2o4gpu_experts_sort(size_t slots, int experts, const int *d_experts, int *d_order, int *d_position,
                                int *d_offsets, void *d_workspace, size_t workspace_bytes, void *stream) {
  if (!experts_ok(experts) || slots > MOST_ROWS || !ints_ok(d_offsets)) return H2O4GPU_KMEANS_EARG;
  if (slots > 0 && (!ints_ok(d_experts) || !ints_ok(d_order) || !ints_ok(d_position))) return H2O4GPU_KMEANS_EARG;
  const size_t need = h2o4gpu_experts_sort_workspace(slots, experts);
  if (need > 0 && (!ints_ok(d_workspace) || workspace_bytes < need)) return H2O4GPU_KMEANS_EARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int buckets = experts + 1;
  const int blocks = sort_blocks(slots) > 0 ? sort_blocks(slots) : 1;
  int *hist = static_cast<int *>(d_workspace);
  // as many wavefronts as counters of their own fit (128 KB): 16 up to 2047 experts, 2 for the most
  int waves = 16;
  while (waves > 1 && (size_t)waves * buckets * sizeof(int) > (128u << 10)) waves >>= 1;
  int bits = 0;
  while ((experts >> bits) != 0) bits++;
  if (blocks > 1) {
    const size_t lds = (size_t)buckets * sizeof(int);
    KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(expert_count_kernel), lds));
    hipLaunchKernelGGL(expert_count_kernel, dim3(blocks), dim3(1024), lds, s, d_experts, (int64_t)slots, experts,
                       hist);
    KM_TRY(launched());
  }
  const size_t lds = ((size_t)waves * buckets + (size_t)waves * WAVE) * sizeof(int);
  KM_TRY(ensure_dynamic_lds(reinterpret_cast<const void *>(expert_place_kernel), lds));
  hipLaunchKernelGGL(expert_place_kernel, dim3(blocks), dim3(waves * WAVE), lds, s, d_experts, (int64_t)slots,
                     experts, bits, hist, blocks, d_order, d_position, d_offsets);
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
    hipLaunchKernelGGL(send_rows_kernel<T>, dim3(grid_of(tokens)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T *>(d_x), (int64_t)x_stride, d_position, (int64_t)tokens, top_k, (int)cols,
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
    auto kernel = weighted ? join_rows_kernel<T, true> : join_rows_kernel<T, false>;
    hipLaunchKernelGGL(kernel, dim3(grid_of(tokens)), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<const T *>(src), (int64_t)src_stride, w, position, (int64_t)tokens, top_k,
                       (int)cols, static_cast<T *>(dst), (int64_t)dst_stride);
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
    hipLaunchKernelGGL(join_backward_kernel<T>, dim3(grid_of(tokens)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), static_cast<const T *>(d_dout), (int64_t)dout_stride,
                       static_cast<const T *>(d_rows), (int64_t)rows_stride, d_weights, d_position, (int64_t)tokens,
                       top_k, (int)cols, static_cast<T *>(d_drows), (int64_t)drows_stride, d_dweights);
    return launched();
  });
}
