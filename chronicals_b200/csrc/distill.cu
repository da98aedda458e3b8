// Distillation from a teacher's top logits.
//
// A row (token) has the student's logits z [V] and up to K entries (index i_k, teacher logit t_k).  With the temperature tau,
//     q = softmax(t / tau) over the row's entries,   Q[i] = the q of all entries of word i,   p = softmax(z / tau) over the vocabulary,
//     row loss = tau^2 sum_i Q[i] (log Q[i] - log p[i]) = tau^2 sum_k q_k (log Q[i_k] - log p[i_k]),   d(row loss) / dz = tau (p - Q).
// An entry takes part when its index lies in [0, V) and its logit is not -inf.  A row takes part when
// it has such an entry and its label, where labels are given, is not the ignored one.  The mean is over the rows that take part.
//
// Two forms.  On logits that a program holds: read once for the loss, once for the gradient, bound by memory.  From hidden
// states and the output weight: the log-sum-exp comes out of the vocabulary product's epilogue (gemm.cu), this file adds the
// teacher's side: the logits of its K words as dot products with gathered weight rows, and their places in the chunks
// of d(logits).
//
// Exponentials are taken in base 2 against a reference that is kept scaled, M = max(z) * log2(e) / tau as it was rounded:
// every term 2^(z log2(e) / tau - M) uses that same M, so its rounding cancels in p and in the loss.
#include <utility>
#include <cooperative_groups.h>
#include "common.cuh"
#include "host_common.h"
#include "logit_rows.cuh"

namespace cg = cooperative_groups;

namespace cb {

constexpr int KD_MAX_K = 4096;                          // entries a row: they are held in shared memory, 12 bytes each
constexpr float KD_LN2 = 0.6931471805599453f;

// A row's entries: indices and logits of either width, labels or none.
struct KdTeacher {
  const void* idx;                                      // int64 or int32 [rows, K], pitch ld_idx
  const void* lg;                                       // fp32 or bf16 [rows, K], pitch ld_lg
  long long ld_idx, ld_lg;
  const long long* labels;                              // [rows] or null
  long long ignore_index;
  int idx64, lg_bf16, K;
  float inv_tau, tau;
};

__device__ __forceinline__ int kd_index(const KdTeacher& t, long long row, int k, int V) {
  const long long i = t.idx64 ? static_cast<const long long*>(t.idx)[row * t.ld_idx + k]
                              : static_cast<const int*>(t.idx)[row * t.ld_idx + k];
  return i >= 0 && i < V ? static_cast<int>(i) : -1;
}
__device__ __forceinline__ float kd_logit(const KdTeacher& t, long long row, int k) {
  return t.lg_bf16 ? __bfloat162float(static_cast<const bf16*>(t.lg)[row * t.ld_lg + k])
                   : static_cast<const float*>(t.lg)[row * t.ld_lg + k];
}

// sums and maxima over a block of up to 32 warps; `red` is shared memory of 32 floats, free again when this returns
__device__ __forceinline__ float kd_block_sum(float v, float* red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  float a = 0.f;
  for (int i = 0; i < nw; ++i) a += red[i];            // the same order in every thread
  __syncthreads();
  return a;
}
__device__ __forceinline__ float kd_block_max(float v, float* red) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  float a = -INFINITY;
  for (int i = 0; i < nw; ++i) a = fmaxf(a, red[i]);
  __syncthreads();
  return a;
}

// Loads a row's entries into shared memory (absent ones with index -1 and logit -inf); true in every thread if the row takes part.
__device__ __forceinline__ bool kd_load(const KdTeacher& t, long long row, int V, int* s_idx, float* s_lg) {
  bool any = false;
  if (t.labels == nullptr || t.labels[row] != t.ignore_index) {
    for (int k = threadIdx.x; k < t.K; k += blockDim.x) {
      int i = kd_index(t, row, k, V);
      float l = -INFINITY;
      if (i >= 0) {
        l = kd_logit(t, row, k) * t.inv_tau;
        if (l == -INFINITY) i = -1;                     // a NaN is an entry, and shows in the loss
      }
      s_idx[k] = i;
      s_lg[k] = l;
      any |= i >= 0;
    }
  }
  return __syncthreads_or(any);
}

// s_lg: logits over tau -> q.  All threads of the block.
__device__ __forceinline__ void kd_softmax(int K, const int* s_idx, float* s_lg, float* red) {
  float m = -INFINITY;
  for (int k = threadIdx.x; k < K; k += blockDim.x) m = fmaxf(m, s_lg[k]);
  m = kd_block_max(m, red);
  float s = 0.f;
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const float e = s_idx[k] >= 0 ? expf(s_lg[k] - m) : 0.f;
    s_lg[k] = e;
    s += e;
  }
  s = kd_block_sum(s, red);
  for (int k = threadIdx.x; k < K; k += blockDim.x) s_lg[k] /= s;
  __syncthreads();
}

// the q of all entries with the index of entry k.  The square of the entries: 4096 rows of 32,000 words, bf16, with 64 / 256 / 1024 / 4096
// entries each take 68 / 101 / 755 / 11,391 us for the loss on held logits (a row's entries are a few dozen as a rule).
__device__ __forceinline__ float kd_merged(int K, const int* s_idx, const float* s_q, int k) {
  const int i = s_idx[k];
  float q = 0.f;
  for (int j = 0; j < K; ++j) q += s_idx[j] == i ? s_q[j] : 0.f;
  return q;
}

// running (M, sum of 2^(v c2 - M)); an all -inf prefix keeps the sum at 0, NaN stays NaN
struct KdAcc {
  float M = -INFINITY, s = 0.f;
  __device__ __forceinline__ static float base(float m) { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void merge(float om, float os) {
    const float nm = fmaxf(M, om), b = base(nm);
    s = s * ex2_approx(M - b) + os * ex2_approx(om - b);
    M = nm;
  }
  template <int N>
  __device__ __forceinline__ void add(const uint4 (&u)[CE_BATCH], const bool (&in)[CE_BATCH], float c2) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i)
      if (in[i]) mx = fmaxf(mx, ce_max<N>(u[i]));
    const float nm = fmaxf(M, mx * c2), b = base(nm);
    float e = 0.f;
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i)
      if (in[i]) {
        float w[N];
        ce_unpack(u[i], w);
#pragma unroll
        for (int j = 0; j < N; ++j) e += ex2_approx(fmaf(w[j], c2, -b));
      }
    s = s * ex2_approx(M - b) + e;
    M = nm;
  }
  __device__ __forceinline__ void add(float v, float c2) {
    const float nm = fmaxf(M, v * c2), b = base(nm);
    s = s * ex2_approx(M - b) + ex2_approx(fmaf(v, c2, -b));
    M = nm;
  }
};

// Loss of a row of held logits.  gridDim.y blocks of a cluster share a row; the first one joins their sums and adds the teacher's
// side.  stats[row] = (M, 1 / sum), or (0, -1) for a row that takes no part; q_out[row, K] = the merged q of each entry.
// 4095 x 151,936 bf16, 64 words a row, a fifth of the rows masked: 176 us, 5.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(CE_THREADS)
kd_logits_kernel(const T* __restrict__ logits, long long ld, int V, const KdTeacher t, float c2, float2* __restrict__ stats,
                 float* __restrict__ q_out, float* __restrict__ loss_rows) {
  constexpr int N = CeVec<T>::N;
  extern __shared__ uint8_t kd_smem[];
  int* s_idx = reinterpret_cast<int*>(kd_smem);
  float* s_q = reinterpret_cast<float*>(s_idx + t.K);
  __shared__ float red[32], sm[CE_THREADS / 32], ss[CE_THREADS / 32];
  __shared__ float part[2][8];
  const long long row = blockIdx.x;
  if (!kd_load(t, row, V, s_idx, s_q)) {               // the same answer in every block of the row
    if (threadIdx.x == 0 && blockIdx.y == 0) {
      stats[row] = make_float2(0.f, -1.f);
      loss_rows[row] = 0.f;
    }
    return;
  }
  // the first block's shared memory may be written only once that block is known to run: everybody arrives here, and whoever
  // writes waits before it does, a row's reading later
  cg::cluster_group cl = cg::this_cluster();
  cg::cluster_group::arrival_token started;
  if (gridDim.y > 1) started = cl.barrier_arrive();
  const T* lp = logits + row * ld;
  const int head = ce_head(lp, V), nvec = (V - head) / N, tail0 = head + nvec * N;
  const uint4* vp = reinterpret_cast<const uint4*>(lp + head);
  const int step = blockDim.x * gridDim.y;
  KdAcc a;
  int c = blockIdx.y * blockDim.x + threadIdx.x;
  uint4 u[CE_BATCH];
  const bool all[CE_BATCH] = {true, true, true, true};
  for (; c + (CE_BATCH - 1) * step < nvec; c += CE_BATCH * step) {
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i) u[i] = vp[c + i * step];
    a.add<N>(u, all, c2);
  }
  if (c < nvec) {                                      // a batch that need not be full
    bool in[CE_BATCH];
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i) {
      in[i] = c + i * step < nvec;
      if (in[i]) u[i] = vp[c + i * step];
    }
    a.add<N>(u, in, c2);
  }
  if (blockIdx.y == 0) {                               // at most N - 1 values at either end
    const int i = static_cast<int>(threadIdx.x);
    if (i < head) a.add(ldf(lp + i), c2);
    if (tail0 + i < V) a.add(ldf(lp + tail0 + i), c2);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, a.M, o), os = __shfl_xor_sync(0xffffffffu, a.s, o);
    a.merge(om, os);
  }
  if ((threadIdx.x & 31) == 0) {
    sm[threadIdx.x >> 5] = a.M;
    ss[threadIdx.x >> 5] = a.s;
  }
  __syncthreads();
  a = KdAcc();
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) a.merge(sm[i], ss[i]);
  if (gridDim.y > 1) {
    cl.barrier_wait(std::move(started));
    if (threadIdx.x == 0) {
      float* dst = cl.map_shared_rank(&part[0][0], 0);
      dst[blockIdx.y] = a.M;
      dst[8 + blockIdx.y] = a.s;
    }
    cl.sync();
    if (blockIdx.y != 0) return;
    a = KdAcc();
    for (unsigned i = 0; i < gridDim.y; ++i) a.merge(part[0][i], part[1][i]);
  }
  kd_softmax(t.K, s_idx, s_q, red);
  const float log2s = log2f(a.s);
  float sum = 0.f;
  for (int k = threadIdx.x; k < t.K; k += blockDim.x) {
    const float q = s_q[k], word = s_idx[k] >= 0 ? kd_merged(t.K, s_idx, s_q, k) : 0.f;
    if (s_idx[k] >= 0 && q != 0.f) sum += q * (logf(word) - (fmaf(ldf(lp + s_idx[k]), c2, -a.M) - log2s) * KD_LN2);
    q_out[row * t.K + k] = word;
  }
  sum = kd_block_sum(sum, red);
  if (threadIdx.x == 0) {
    stats[row] = make_float2(a.M, 1.f / a.s);
    loss_rows[row] = t.tau * t.tau * sum;
  }
}

// d(loss) / dz of held logits.  A block takes a stretch of a row: the softmax's part for every value, then the values of the
// teacher's words that lie in it once more, with theirs.  At the size above: 367 us, 6.1 TB/s.
template <typename T>
__global__ void __launch_bounds__(CE_THREADS)
kd_logits_grad_kernel(const T* __restrict__ logits, T* __restrict__ dlogits, long long ld, long long ldd, int V, const KdTeacher t,
                      float c2, const float2* __restrict__ stats, const float* __restrict__ q, const float* __restrict__ gout,
                      const float* __restrict__ n_rows, const float* __restrict__ grows) {
  constexpr int N = CeVec<T>::N;
  const long long row = blockIdx.x;
  const T* lp = logits + row * ld;
  T* dp = dlogits + row * ldd;
  const float2 st = stats[row];
  const bool valid = !(st.y == -1.f);
  float g = 0.f;
  if (gout != nullptr) g += n_rows != nullptr ? gout[0] / fmaxf(n_rows[0], 1.f) : gout[0];
  if (grows != nullptr) g += grows[row];
  g *= t.tau;
  const float gs = st.y * g;
  const auto e2 = [&](float v) {                       // fp32 results want more than the approximation's 22 bits
    const float x = fmaf(v, c2, -st.x);
    return sizeof(T) == 2 ? ex2_approx(x) : exp2f(x);
  };
  const int head = ce_head(lp, V), nvec = (V - head) / N;                 // the same of both rows
  const uint4* vp = reinterpret_cast<const uint4*>(lp + head);
  uint4* wp = reinterpret_cast<uint4*>(dp + head);
  // this block's stretch: vectors [v0, v1), with the values before the first vector and after the last at the ends
  const int y = blockIdx.y, per = (nvec + gridDim.y - 1) / gridDim.y;
  const int v0 = min(nvec, y * per), v1 = min(nvec, v0 + per);
  const bool lowest = y == 0, highest = y == static_cast<int>(gridDim.y) - 1;
  const int c0 = lowest ? 0 : head + v0 * N, c1 = highest ? V : head + v1 * N;
  const int tail0 = head + nvec * N, step = blockDim.x;
  if (!valid) {
    for (int v = v0 + threadIdx.x; v < v1; v += step) wp[v] = make_uint4(0u, 0u, 0u, 0u);
    if (lowest) for (int c = threadIdx.x; c < head; c += step) stf(dp + c, 0.f);
    if (highest) for (int c = tail0 + threadIdx.x; c < V; c += step) stf(dp + c, 0.f);
    return;
  }
  for (int v = v0 + threadIdx.x; v < v1; v += CE_BATCH * step) {
    uint4 u[CE_BATCH];
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i)
      if (v + i * step < v1) u[i] = vp[v + i * step];
#pragma unroll
    for (int i = 0; i < CE_BATCH; ++i)
      if (v + i * step < v1) {
        float w[N];
        ce_unpack(u[i], w);
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = e2(w[j]) * gs;
        wp[v + i * step] = ce_pack(w);
      }
  }
  if (lowest) for (int c = threadIdx.x; c < head; c += step) stf(dp + c, e2(ldf(lp + c)) * gs);
  if (highest) for (int c = tail0 + threadIdx.x; c < V; c += step) stf(dp + c, e2(ldf(lp + c)) * gs);
  __syncthreads();                                     // the values above are written before those below
  for (int k = threadIdx.x; k < t.K; k += step) {
    const int i = kd_index(t, row, k, V);
    if (i >= c0 && i < c1) {
      const float qk = q[row * t.K + k];
      if (qk != 0.f) stf(dp + i, (e2(ldf(lp + i)) * st.y - qk) * g);   // every entry of one index writes the same value
    }
  }
}

// The factor c of d(logits) as 2^k times a rest in [1, 2).  Products of bf16 d(logits) are formed with 2^k and their results multiplied by
// the rest in 32 bits: at a teacher's only word p - Q is close to -1 in every row, and c would be rounded the same way in all of them (by
// up to 2^-8, which no sum averages out).
__device__ __forceinline__ float kd_unit(float c, float& rest) {
  int e;
  const float m = frexpf(c, &e);
  const bool whole = c != 0.f && isfinite(c);
  rest = whole ? 2.f * m : 1.f;
  return whole ? ldexpf(1.f, e - 1) : c;
}

// d(loss) / dz of fp32 logits as bf16, for the products that follow; with `lo` also what the rounding left out, in a second set of rows
// (the products of few tokens have room for twice as many rows, and add the two in 32 bits).  Rows of both on 16-byte boundaries,
// their pitches multiples of 8; a thread takes 8 values.  Blocks and words as in the kernel above.  With `rest` the factor is a power of
// two, and rest[0] what is left of it.  1021 x 151,936, a fifth of the rows
// masked: 131 us, 6.2 TB/s.
__global__ void __launch_bounds__(CE_THREADS)
kd_logits_grad_split_kernel(const float* __restrict__ logits, bf16* __restrict__ hi, bf16* __restrict__ lo, long long ld, long long ldg,
                            int V, const KdTeacher t, float c2, const float2* __restrict__ stats, const float* __restrict__ q,
                            const float* __restrict__ gout, const float* __restrict__ n_rows, const float* __restrict__ grows,
                            float* __restrict__ rest) {
  const long long row = blockIdx.x;
  const float* lp = logits + row * ld;
  bf16* hp = hi + row * ldg;
  bf16* rp = lo != nullptr ? lo + row * ldg : nullptr;
  const float2 st = stats[row];
  float g = 0.f;
  if (gout != nullptr) g += n_rows != nullptr ? gout[0] / fmaxf(n_rows[0], 1.f) : gout[0];
  if (grows != nullptr) g += grows[row];
  g *= t.tau;
  if (rest != nullptr) {
    float left;
    g = kd_unit(g, left);
    if (blockIdx.y == 0 && row == 0 && threadIdx.x == 0) rest[0] = left;
  }
  const bool valid = !(st.y == -1.f);
  const float gs = valid ? st.y * g : 0.f;
  const auto put = [&](int i, float v) {
    hp[i] = __float2bfloat16(v);
    if (rp != nullptr) rp[i] = __float2bfloat16(v - __bfloat162float(hp[i]));
  };
  const int nvec = V / 8, y = blockIdx.y, per = (nvec + gridDim.y - 1) / gridDim.y;
  const int v0 = min(nvec, y * per), v1 = min(nvec, v0 + per);
  const bool highest = y == static_cast<int>(gridDim.y) - 1;
  const int c0 = v0 * 8, c1 = highest ? V : v1 * 8;
  for (int v = v0 + threadIdx.x; v < v1; v += blockDim.x) {
    uint4 h = make_uint4(0u, 0u, 0u, 0u), l = h;
    if (valid) {
      const float4 a = reinterpret_cast<const float4*>(lp)[2 * v], b = reinterpret_cast<const float4*>(lp)[2 * v + 1];
      float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = exp2f(fmaf(w[j], c2, -st.x)) * gs;
      h = pack8(w);
      unpack8(h, f);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] -= f[j];
      l = pack8(w);
    }
    reinterpret_cast<uint4*>(hp)[v] = h;
    if (rp != nullptr) reinterpret_cast<uint4*>(rp)[v] = l;
  }
  if (highest)
    for (int c = nvec * 8 + threadIdx.x; c < V; c += blockDim.x) put(c, valid ? exp2f(fmaf(lp[c], c2, -st.x)) * gs : 0.f);
  if (!valid) return;
  __syncthreads();                                     // the values above are written before those below
  for (int k = threadIdx.x; k < t.K; k += blockDim.x) {
    const int i = kd_index(t, row, k, V);
    if (i >= c0 && i < c1) {
      const float qk = q[row * t.K + k];
      if (qk != 0.f) put(i, (exp2f(fmaf(lp[i], c2, -st.x)) * st.y - qk) * g);          // every entry of one index writes the same value
    }
  }
}

// loss = mean (or sum) of the rows' losses, n_rows = rows that take part; with gscale also 1 for each of them and 0 for the others.  stats.y == -1 marks the rows that take no part.  One block, a fixed order.
__global__ void __launch_bounds__(1024)
kd_finalize_kernel(const float* __restrict__ loss_rows, const float2* __restrict__ stats, long long rows, int mean,
                   float* __restrict__ loss, float* __restrict__ n_rows, float* __restrict__ gscale) {
  __shared__ float red[32];
  float sum = 0.f, cnt = 0.f;
  for (long long i = threadIdx.x; i < rows; i += blockDim.x) {
    const bool on = !(stats[i].y == -1.f);
    sum += on ? loss_rows[i] : 0.f;
    cnt += on ? 1.f : 0.f;
  }
  sum = kd_block_sum(sum, red);
  cnt = kd_block_sum(cnt, red);
  if (threadIdx.x == 0) {
    loss[0] = mean ? sum / fmaxf(cnt, 1.f) : sum;
    n_rows[0] = cnt;
  }
  if (gscale != nullptr)
    for (long long i = threadIdx.x; i < rows; i += blockDim.x) gscale[i] = stats[i].y == -1.f ? 0.f : 1.f;
}

// ------------------------------------------------------------------ from hidden states and the output weight
// idle[b] = 1 where none of the rows [128 b, 128 b + 128) takes part: the vocabulary products leave such blocks out (prompts are often
// long, and masked).
__global__ void __launch_bounds__(128)
kd_idle_kernel(const KdTeacher t, int V, long long M, int* __restrict__ idle) {
  const long long row = blockIdx.x * 128LL + threadIdx.x;
  bool on = false;
  if (row < M && (t.labels == nullptr || t.labels[row] != t.ignore_index))
    for (int k = 0; k < t.K && !on; ++k) on = kd_index(t, row, k, V) >= 0 && kd_logit(t, row, k) * t.inv_tau != -INFINITY;
  const int any = __syncthreads_or(on);
  if (threadIdx.x == 0) idle[blockIdx.x] = any ? 0 : 1;
}

// One block a row, after the vocabulary product has left its partial maxima and sums: the row's log-sum-exp, the student's logits of
// the teacher's words (dot products of the hidden row, kept in shared memory, with gathered weight rows: KD_DOTS rows a warp at
// a time, so that as many loads are in flight), the loss, and coef[row, K] = p - q, what d(logits) holds at those words.
// Bound by the gathers: K weight rows a token.  8192 x 896, 64 words a row, a fifth of the rows masked: 152 us (5 TB/s, part of it from
// L2), 178 after the products with their clock; 4 rows at a time 196, 8 278, 256 threads 181 (against 152).
constexpr int KD_DOTS = 2, KD_ROW_THREADS = 128;

__global__ void __launch_bounds__(KD_ROW_THREADS)
kd_linear_rows_kernel(const bf16* __restrict__ hidden, long long ldh, const bf16* __restrict__ weight, long long ldw, int H, int V,
                      int M, const float* __restrict__ part_m, const float* __restrict__ part_s, int n_splits, const KdTeacher t,
                      float c2, float* __restrict__ lse, float2* __restrict__ stats, float* __restrict__ coef,
                      int* __restrict__ words, float* __restrict__ loss_rows) {
  extern __shared__ uint8_t kd_smem[];
  uint4* s_h = reinterpret_cast<uint4*>(kd_smem);      // H / 8 vectors
  int* s_idx = reinterpret_cast<int*>(s_h + H / 8);
  float* s_q = reinterpret_cast<float*>(s_idx + t.K);
  float* s_z = s_q + t.K;                              // the student's logits
  __shared__ float red[32];
  const long long row = blockIdx.x;
  if (!kd_load(t, row, V, s_idx, s_q)) {               // its partial sums may not exist
    if (threadIdx.x == 0) {
      stats[row] = make_float2(0.f, -1.f);
      loss_rows[row] = 0.f;
      lse[row] = 1e30f;                                // probabilities of zero, whatever the logits
    }
    return;
  }
  KdAcc a;
  {
    float m = -INFINITY;
    for (int i = threadIdx.x; i < n_splits; i += blockDim.x) m = fmaxf(m, part_m[static_cast<long long>(i) * M + row]);
    m = kd_block_max(m, red);
    a.M = m * c2;
    float s = 0.f;
    for (int i = threadIdx.x; i < n_splits; i += blockDim.x) {
      const long long o = static_cast<long long>(i) * M + row;
      if (part_m[o] > -INFINITY) s += part_s[o] * ex2_approx(part_m[o] * c2 - a.M);
    }
    a.s = kd_block_sum(s, red);
  }
  const float log2s = log2f(a.s);
  if (threadIdx.x == 0) lse[row] = (a.M + log2s) * KD_LN2;
  const int nv = H / 8, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) s_h[i] = reinterpret_cast<const uint4*>(hidden + row * ldh)[i];
  __syncthreads();
  for (int k0 = warp * KD_DOTS; k0 < t.K; k0 += nw * KD_DOTS) {
    const uint4* w[KD_DOTS];
    float acc[KD_DOTS];
#pragma unroll
    for (int d = 0; d < KD_DOTS; ++d) {
      const int i = k0 + d < t.K ? s_idx[k0 + d] : -1;
      w[d] = i >= 0 ? reinterpret_cast<const uint4*>(weight + i * ldw) : nullptr;
      acc[d] = 0.f;
    }
    for (int v = lane; v < nv; v += 32) {
      uint4 u[KD_DOTS];
#pragma unroll
      for (int d = 0; d < KD_DOTS; ++d) u[d] = w[d] != nullptr ? w[d][v] : make_uint4(0u, 0u, 0u, 0u);
      float h[8];
      unpack8(s_h[v], h);
#pragma unroll
      for (int d = 0; d < KD_DOTS; ++d) {
        float x[8];
        unpack8(u[d], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[d] = fmaf(h[j], x[j], acc[d]);
      }
    }
#pragma unroll
    for (int d = 0; d < KD_DOTS; ++d) {
      const float z = warp_sum(acc[d]);
      if (lane == 0 && k0 + d < t.K) s_z[k0 + d] = z;
    }
  }
  __syncthreads();
  kd_softmax(t.K, s_idx, s_q, red);
  float sum = 0.f;
  for (int k = threadIdx.x; k < t.K; k += blockDim.x) {
    float d = 0.f;
    if (s_idx[k] >= 0) {
      const float q = s_q[k], word = kd_merged(t.K, s_idx, s_q, k);
      const float l2 = fmaf(s_z[k], c2, -a.M) - log2s;                   // log2 p
      if (q != 0.f) sum += q * (logf(word) - l2 * KD_LN2);
      d = exp2f(l2) - word;
    }
    coef[row * t.K + k] = d;
    words[row * t.K + k] = s_idx[k];
  }
  sum = kd_block_sum(sum, red);
  if (threadIdx.x == 0) {
    stats[row] = make_float2(a.M, 1.f / a.s);
    loss_rows[row] = t.tau * t.tau * sum;
  }
}

// The factor of d(logits) from hidden states: unit[0] = its power of two, unit[1] = the rest.  One thread.
__global__ void kd_unit_kernel(const float* __restrict__ gout, const float* __restrict__ n_rows, float tau, float* __restrict__ unit) {
  float left;
  unit[0] = kd_unit(tau * gout[0] / (n_rows != nullptr ? fmaxf(n_rows[0], 1.f) : 1.f), left);
  unit[1] = left;
}

// out = bf16(x times the rest): d(hidden) summed in 32 bits; n8 times 8 values
__global__ void __launch_bounds__(256)
kd_cast_kernel(const float4* __restrict__ x, uint4* __restrict__ out, long long n8, const float* __restrict__ rest) {
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= n8) return;
  const float r = rest != nullptr ? rest[0] : 1.f;
  const float4 a = x[2 * i], b = x[2 * i + 1];
  const float w[8] = {a.x * r, a.y * r, a.z * r, a.w * r, b.x * r, b.y * r, b.z * r, b.w * r};
  out[i] = pack8(w);
}

// G[row, i - c0] = gscale gout (p - q) for the teacher's words i in [c0, c0 + Vc), over the softmax's part that the product left.
// words [M, K]: -1 for an absent entry.  A warp a row: every chunk looks at every entry, so the entries are read as plainly as can be
// (8192 rows of 64 words, 19 chunks: 5 us each, as long as a launch).
__global__ void __launch_bounds__(CE_THREADS)
kd_place_kernel(bf16* __restrict__ G, long long ldg, int c0, int Vc, long long M, int K, const int* __restrict__ words,
                const float* __restrict__ coef, const float* __restrict__ gscale, const float* __restrict__ gout) {
  const long long row = blockIdx.x * static_cast<long long>(CE_THREADS / 32) + (threadIdx.x >> 5);
  if (row >= M) return;
  const float gs = gscale[row];
  if (gs == 0.f) return;                               // a row that takes no part has no words either
  for (int k = threadIdx.x & 31; k < K; k += 32) {
    const int w = words[row * K + k], i = w - c0;
    if (w >= 0 && i >= 0 && i < Vc) G[row * ldg + i] = __float2bfloat16(coef[row * K + k] * gs * gout[0]);   // one index, one value
  }
}

}  // namespace cb

// =========================================================================================== host side
namespace {

// false: a size that the kernels do not take
bool kd_teacher(cb::KdTeacher* t, const void* idx, long long ld_idx, int idx64, const void* lg, long long ld_lg, int lg_bf16, int K,
                const long long* labels, long long ignore_index, float tau) {
  if (K < 1 || K > cb::KD_MAX_K || !(tau > 0.f)) return false;
  t->idx = idx; t->ld_idx = ld_idx; t->idx64 = idx64;
  t->lg = lg; t->ld_lg = ld_lg; t->lg_bf16 = lg_bf16; t->K = K;
  t->labels = labels; t->ignore_index = ignore_index;
  t->tau = tau; t->inv_tau = 1.f / tau;
  return true;
}
float kd_scale(float tau) { return static_cast<float>(1.4426950408889634 / static_cast<double>(tau)); }

}  // namespace

extern "C" {

int cb_kd_max_entries() { return cb::KD_MAX_K; }

// Held logits: stats [rows, 2], q [rows, K], loss_rows [rows]; loss: their mean (or sum), n_rows: the rows that take part.
int cb_kd_logits(const void* logits, long long rows, long long ld, int V, int is_bf16, const void* idx, long long ld_idx, int idx64,
                 const void* lg, long long ld_lg, int lg_bf16, int K, const long long* labels, long long ignore_index, float tau,
                 int mean, float* stats, float* q, float* loss_rows, float* loss, float* n_rows, void* stream) {
  cb::KdTeacher t;
  if (rows <= 0 || rows > 0x7fffffffLL || V <= 0 || !kd_teacher(&t, idx, ld_idx, idx64, lg, ld_lg, lg_bf16, K, labels, ignore_index, tau))
    return -1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  const int split = cbhost::ce_cluster(rows, V / (is_bf16 ? 8 : 4));
  cfg.gridDim = dim3(static_cast<unsigned>(rows), split);
  cfg.blockDim = dim3(cbhost::ce_threads(rows, V, is_bf16));
  cfg.dynamicSmemBytes = static_cast<size_t>(K) * 8;
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = split;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  const float c2 = kd_scale(tau);
  float2* st = reinterpret_cast<float2*>(stats);
  const cudaError_t e = is_bf16 ? cudaLaunchKernelEx(&cfg, cb::kd_logits_kernel<cb::bf16>, static_cast<const cb::bf16*>(logits), ld, V,
                                                     t, c2, st, q, loss_rows)
                                : cudaLaunchKernelEx(&cfg, cb::kd_logits_kernel<float>, static_cast<const float*>(logits), ld, V, t, c2,
                                                     st, q, loss_rows);
  if (e != cudaSuccess) return static_cast<int>(e);
  cb::kd_finalize_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(loss_rows, st, rows, mean, loss, n_rows, nullptr);
  return static_cast<int>(cudaGetLastError());
}

// Rows of dlogits start at the same distance from a 16-byte boundary as those of logits.
// gout: gradient of the reduced loss (or null), over n_rows[0] for a mean (null: a sum); grows [rows]: of the rows' losses (or null)
int cb_kd_logits_grad(const void* logits, void* dlogits, long long rows, long long ld, long long ldd, int V, int is_bf16,
                      const void* idx, long long ld_idx, int idx64, const void* lg, long long ld_lg, int lg_bf16, int K,
                      const long long* labels, long long ignore_index, float tau, const float* stats, const float* q,
                      const float* gout, const float* n_rows, const float* grows, void* stream) {
  cb::KdTeacher t;
  if (rows <= 0 || rows > 0x7fffffffLL || V <= 0 || !kd_teacher(&t, idx, ld_idx, idx64, lg, ld_lg, lg_bf16, K, labels, ignore_index, tau))
    return -1;
  const long long apart = (ldd - ld) * (is_bf16 ? 2 : 4);
  if (((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15) != 0 || (rows > 1 && apart % 16 != 0)) return -1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows), cbhost::ce_split(rows, V));
  const int threads = cbhost::ce_threads(rows, V, is_bf16);
  const float c2 = kd_scale(tau);
  const float2* st = reinterpret_cast<const float2*>(stats);
  if (is_bf16)
    cb::kd_logits_grad_kernel<cb::bf16><<<grid, threads, 0, s>>>(static_cast<const cb::bf16*>(logits), static_cast<cb::bf16*>(dlogits),
                                                                 ld, ldd, V, t, c2, st, q, gout, n_rows, grows);
  else
    cb::kd_logits_grad_kernel<float><<<grid, threads, 0, s>>>(static_cast<const float*>(logits), static_cast<float*>(dlogits), ld, ldd,
                                                              V, t, c2, st, q, gout, n_rows, grows);
  return static_cast<int>(cudaGetLastError());
}

// fp32 logits -> their gradient as bf16 hi [rows, V], and (lo not null) what the rounding left out; rest [1] or null
int cb_kd_logits_grad_split(const float* logits, void* hi, void* lo, long long rows, long long ld, long long ldg, int V, const void* idx,
                            long long ld_idx, int idx64, const void* lg, long long ld_lg, int lg_bf16, int K, const long long* labels,
                            long long ignore_index, float tau, const float* stats, const float* q, const float* gout,
                            const float* n_rows, const float* grows, float* rest, void* stream) {
  cb::KdTeacher t;
  if (rows <= 0 || rows > 0x7fffffffLL || V <= 0 || ld % 8 != 0 || ldg % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(hi) | reinterpret_cast<uintptr_t>(lo)) & 15) != 0 ||
      !kd_teacher(&t, idx, ld_idx, idx64, lg, ld_lg, lg_bf16, K, labels, ignore_index, tau))
    return -1;
  int split = 1;                                        // blocks a row: until the chip is full, or a block has 2048 values
  while (split < 64 && rows * split < 4LL * cbhost::num_sms() && V / (2 * split) >= 2048) split *= 2;
  cb::kd_logits_grad_split_kernel<<<dim3(static_cast<unsigned>(rows), split), cb::CE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
      logits, static_cast<cb::bf16*>(hi), static_cast<cb::bf16*>(lo), ld, ldg, V, t, kd_scale(tau), reinterpret_cast<const float2*>(stats), q,
      gout, n_rows, grows, rest);
  return static_cast<int>(cudaGetLastError());
}

// From hidden states, first of all: idle [ceil(M / 128)]
int cb_kd_idle(const void* idx, long long ld_idx, int idx64, const void* lg, long long ld_lg, int lg_bf16, int K, const long long* labels,
               long long ignore_index, float tau, int V, int M, int* idle, void* stream) {
  cb::KdTeacher t;
  if (M <= 0 || V <= 0 || !kd_teacher(&t, idx, ld_idx, idx64, lg, ld_lg, lg_bf16, K, labels, ignore_index, tau)) return -1;
  cb::kd_idle_kernel<<<(M + 127) / 128, 128, 0, static_cast<cudaStream_t>(stream)>>>(t, V, M, idle);
  return static_cast<int>(cudaGetLastError());
}

// From hidden states, after cb_cce_forward_t: part_m / part_s [n_splits, M].  lse, loss_rows, gscale [M], stats [M, 2], coef and
// words [M, K], loss and n_rows as above.
int cb_kd_linear_rows(const void* hidden, long long ldh, const void* weight, long long ldw, int H, int V, int M, const float* part_m,
                      const float* part_s, int n_splits, const void* idx, long long ld_idx, int idx64, const void* lg, long long ld_lg,
                      int lg_bf16, int K, const long long* labels, long long ignore_index, float tau, int mean, float* lse,
                      float* stats, float* coef, int* words, float* loss_rows, float* loss, float* n_rows, float* gscale, void* stream) {
  cb::KdTeacher t;
  if (M <= 0 || V <= 0 || H <= 0 || H % 8 != 0 || ldh % 8 != 0 || ldw % 8 != 0 ||
      ((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight)) & 15) != 0 ||
      !kd_teacher(&t, idx, ld_idx, idx64, lg, ld_lg, lg_bf16, K, labels, ignore_index, tau))
    return -1;
  const int smem = H * 2 + K * 12;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (smem > 227 * 1024 - 1024) return -1;
  if (smem > 48 * 1024) CB_CHECK_CUDA(cudaFuncSetAttribute(cb::kd_linear_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024));
  float2* st = reinterpret_cast<float2*>(stats);
  cb::kd_linear_rows_kernel<<<M, cb::KD_ROW_THREADS, smem, s>>>(
      static_cast<const cb::bf16*>(hidden), ldh, static_cast<const cb::bf16*>(weight), ldw, H, V, M, part_m, part_s, n_splits, t,
      kd_scale(tau), lse, st, coef, words, loss_rows);
  CB_CHECK_CUDA(cudaGetLastError());
  cb::kd_finalize_kernel<<<1, 1024, 0, s>>>(loss_rows, st, M, mean, loss, n_rows, gscale);
  return static_cast<int>(cudaGetLastError());
}

// unit [2] for the backward pass from hidden states; n_rows null: a sum
int cb_kd_unit(const float* gout, const float* n_rows, float tau, float* unit, void* stream) {
  cb::kd_unit_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(gout, n_rows, tau, unit);
  return static_cast<int>(cudaGetLastError());
}

// out [n] bf16 = x [n] fp32 times rest[0] (null: 1); n a multiple of 8
int cb_kd_cast(const float* x, void* out, long long n, const float* rest, void* stream) {
  if (n <= 0 || n % 8 != 0 || ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) != 0) return -1;
  const long long blocks = (n / 8 + 255) / 256;
  if (blocks > 0x7fffffffLL) return -1;
  cb::kd_cast_kernel<<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const float4*>(x), static_cast<uint4*>(out), n / 8, rest);
  return static_cast<int>(cudaGetLastError());
}

// The teacher's words in a chunk [c0, c0 + Vc) of d(logits), as cb_kd_linear_rows left them
int cb_kd_place(void* G, long long ldg, int c0, int Vc, int M, int K, const int* words, const float* coef, const float* gscale,
                const float* gout, void* stream) {
  if (M <= 0 || Vc <= 0 || K < 1) return -1;
  constexpr int rows = cb::CE_THREADS / 32;
  cb::kd_place_kernel<<<(M + rows - 1) / rows, cb::CE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<cb::bf16*>(G), ldg, c0, Vc, M, K, words, coef, gscale, gout);
  return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
