// Rows of logits, as the losses on held logits read and write them: 16-byte vectors between the first and the last 16-byte
// boundary of a row, the values outside them one by one, and the number of blocks and threads that a row is given.
#pragma once
#include "common.cuh"
#include "host_common.h"

namespace cb {

constexpr int CE_THREADS = 256;
constexpr int CE_BATCH = 4;

template <typename T>
struct CeVec {
  static constexpr int N = 16 / sizeof(T);
};
__device__ __forceinline__ void ce_unpack(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void ce_unpack(const uint4& u, float (&f)[8]) { unpack8(u, f); }
__device__ __forceinline__ uint4 ce_pack(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 ce_pack(const float (&f)[8]) { return pack8(f); }
__device__ __forceinline__ float ldf(const float* p) { return *p; }
__device__ __forceinline__ float ldf(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void stf(float* p, float v) { *p = v; }
__device__ __forceinline__ void stf(bf16* p, float v) { *p = __float2bfloat16(v); }

// values in front of the first 16-byte boundary of a row (at most V)
template <typename T>
__device__ __forceinline__ int ce_head(const T* p, int V) {
  const int h = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  return h < V ? h : V;
}

template <int N>
__device__ __forceinline__ float ce_max(const uint4& u) {
  if (N == 4) return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  const bf162* h = reinterpret_cast<const bf162*>(&u);
  const float2 f = __bfloat1622float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
  return fmaxf(f.x, f.y);
}

}  // namespace cb

namespace cbhost {

// Blocks that share one row of logits.  In the gradient, one is enough once the rows alone fill the chip (four blocks an SM); with
// fewer, a row is cut in 2, 4 or 8 as long as every piece keeps 4096 values.
inline int ce_split(long long rows, int V) {
  int split = 1;
  while (split < 8 && rows * split < 4LL * num_sms() && V / (2 * split) >= 4096) split *= 2;
  return split;
}
// In the forward pass, where a row is `nvec` 16-byte vectors, they form a cluster (a portable one has 8 at most) and meeting costs
// about a microsecond: long rows as above in pieces of 2048 vectors; very long ones in pieces of 4096 also when there are many,
// since rows that are masked leave the rest unevenly spread over one round of blocks; or rows so few that they leave half the
// SMs without a block.  Measured, bf16, one / two / four blocks a row: 16 x 32,000 6.2 / 5.4 / 4.4 us, 200 x 50,257 (one: 11 and
// more) 9.7 / 10.4, 400 x 16,384 6.3 / 8.1, 100 x 8192 3.5 / 4.4; 2047 x 151,936 fp32, a fifth of the rows masked, 173 / 145;
// 1000 x 100,000 bf16, half of them, 47 / 31.  Not with rows
// for more than one round: 4095 x 151,936 bf16, a fifth masked (distillation), 175 / 190 / 217.
inline int ce_cluster(long long rows, int nvec) {
  int split = 1;
  while (split < 8 && ((rows * split < 4LL * num_sms() && nvec / (2 * split) >= 2048) ||
                       (rows * split < 24LL * num_sms() && nvec / (2 * split) >= 4096) ||
                       (2 * rows * split <= num_sms() && nvec / 3 >= 1024 && nvec / (2 * split) >= 512)))
    split *= 2;
  return split;
}
// Threads of a block of a row of logits: with rows enough to fill the chip (four blocks an SM) as many as have a whole batch of
// vectors each, since a block of 256 for a row of a few kilobytes spends most of its time on reductions between threads without
// data (20,000 x 1000 bf16: forward 58 us with 256 threads, 22 with 32); with fewer rows, a thread a vector.
inline int ce_threads(long long rows, int V, int is_bf16) {
  const int nvec = V / (is_bf16 ? 8 : 4) + 1, each = rows > 4LL * num_sms() ? cb::CE_BATCH : 1;
  const int t = ((nvec + each - 1) / each + 31) / 32 * 32;
  return t < cb::CE_THREADS ? t : cb::CE_THREADS;
}

}  // namespace cbhost
