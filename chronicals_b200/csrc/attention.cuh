// What the attention kernels share: their arguments, the tiles of the windowed forms, and the operand images in shared memory.
#pragma once
#include "common.cuh"

namespace cb {

constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
  int T, hq, hk, n_docs;
  const int* cu;        // [n_docs + 1]
  float scale;
  bf16* O;              // [T, hq, D], row pitch ldo
  long long ldo;
  float* lse;           // [hq, T]
  // backward
  const float* delta;   // [hq, T]  rowsum(dO * O)
  float* dq_acc;        // [T, hq, D] fp32, zero-initialised; accumulated with red.add
  float* dk_part;       // [T, hk, D] fp32, zero-initialised; accumulated with red.add over the group's query heads
  float* dv_part;
  int* status;
  int o_tma;            // forward: a tensor map over O exists, whole blocks may leave by TMA store
  // windowed forms: a query sees the last `window` keys of its document, its own among them, and the document's first `sinks`
  int window, sinks;
  bf16* o_lo;           // forward, [T, hq, D] without gaps or null: O less its rounding to bf16, rounded itself (for delta)
  int sink_run;         // backward: query blocks per CTA of a key block that holds sinks
};

// The tile of a windowed kernel: CTA b's, document by document, the weights being all but equal (a window's worth of blocks).
// Forward, one tile per query block, the last block of a document first.  Backward, one per key block; a key block that holds sinks
// is seen by every later query of its document, and its query blocks are shared out over CTAs in runs of a.sink_run, which come
// first in their document.  blk: the block of the tile, run: of which run (-1: a key block without sinks).
template <bool BWD>
__device__ __forceinline__ bool locate_window_tile(const AttnArgs& a, int b, int& start, int& len, int& nblk, int& blk, int& run,
                                                   int* beyond = nullptr) {
  const int lane = threadIdx.x & 31;
  const int with_sinks = BWD ? (a.sinks + 127) >> 7 : 0;
  for (int d0 = 0; d0 < a.n_docs; d0 += 32) {
    const int d = d0 + lane;
    int st = 0, ln = 0;
    if (d < a.n_docs) {
      st = a.cu[d];
      ln = a.cu[d + 1] - st;
    }
    const int nb = (ln + 127) >> 7, ns = min(nb, with_sinks);
    const int runs = BWD ? (nb + a.sink_run - 1) / a.sink_run : 0;
    const int mine = nb - ns + ns * runs;
    int upto = mine;                                   // tiles of the documents up to mine
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned m = __ballot_sync(0xffffffffu, b < upto);
    if (m != 0) {
      const int src = __ffs(m) - 1;
      const int at = b - __shfl_sync(0xffffffffu, upto - mine, src);
      start = __shfl_sync(0xffffffffu, st, src);
      len = __shfl_sync(0xffffffffu, ln, src);
      nblk = __shfl_sync(0xffffffffu, nb, src);
      const int n_s = __shfl_sync(0xffffffffu, ns, src), n_r = __shfl_sync(0xffffffffu, runs, src);
      if (!BWD) {
        blk = nblk - 1 - at;
        run = -1;
      } else if (at < n_s * n_r) {
        blk = at % n_s;
        run = at / n_s;
      } else {
        blk = at - n_s * n_r + n_s;
        run = -1;
      }
      return true;
    }
    b -= __shfl_sync(0xffffffffu, upto, 31);
  }
  if (beyond != nullptr) *beyond = b;                  // index among the CTAs past the last tile
  return false;
}

// The query blocks [first, first + count) that key block `jb` of a document of nblk blocks meets, or those of its run
__device__ __forceinline__ void window_query_blocks(const AttnArgs& a, int jb, int run, int nblk, int& first, int& count) {
  const int lo = run < 0 ? jb : max(jb, run * a.sink_run);
  const int hi = run < 0 ? min(nblk, ((jb * 128 + 127 + a.window - 1) >> 7) + 1) : min(nblk, (run + 1) * a.sink_run);
  first = lo;
  count = hi - lo;
}

// The grid holds at least ceil((T - cu[n_docs]) / 128) CTAs past the last tile (per head).  In the forward
// kernels they write the zeros of the padding rows at or after cu[n_docs], 128 rows x D columns each, so the
// caller need not clear the output first.
template <int D>
__device__ __forceinline__ void zero_padding_rows(const AttnArgs& a, int beyond, int h) {
  const int valid = a.cu[a.n_docs];
  const long long row0 = static_cast<long long>(valid) + static_cast<long long>(beyond) * 128;
  constexpr int CH = D / 8;                            // 16-byte chunks per row of one head
  for (int i = threadIdx.x; i < 128 * CH; i += blockDim.x) {
    const long long t = row0 + i / CH;
    if (t < a.T) reinterpret_cast<uint4*>(a.O + t * a.ldo + static_cast<long long>(h) * D)[i % CH] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// store 32 consecutive values of thread-row r as bf16 into a [128 x 128] operand image made of two
// 64-column panels of 16 KB, 128-byte rows, 16-byte chunks XOR-swizzled by (row & 7)
__device__ __forceinline__ void store_row_chunk32(uint8_t* base, int r, int c32, const float (&v)[32]) {
  const int panel = c32 >> 1;                 // chunks 0,1 -> panel 0 ; 2,3 -> panel 1
  uint8_t* row = base + panel * 16384 + r * 128;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int cc = (c32 & 1) * 4 + q;         // 16-byte chunk index within the 128-byte row
    uint4 u;
    u.x = pack_bf16x2(v[8 * q + 0], v[8 * q + 1]);
    u.y = pack_bf16x2(v[8 * q + 2], v[8 * q + 3]);
    u.z = pack_bf16x2(v[8 * q + 4], v[8 * q + 5]);
    u.w = pack_bf16x2(v[8 * q + 6], v[8 * q + 7]);
    *reinterpret_cast<uint4*>(row + ((cc ^ (r & 7)) << 4)) = u;
  }
}

// the same for 32 values already packed as bf16 pairs
__device__ __forceinline__ void store_row_chunk32_packed(uint8_t* base, int r, int c32, const uint32_t (&v)[16]) {
  const int panel = c32 >> 1;
  uint8_t* row = base + panel * 16384 + r * 128;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int cc = (c32 & 1) * 4 + q;
    *reinterpret_cast<uint4*>(row + ((cc ^ (r & 7)) << 4)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  }
}

// the same for 16 packed values
__device__ __forceinline__ void store_row_chunk16_packed(uint8_t* base, int r, int c16, const uint32_t (&v)[8]) {
  uint8_t* row = base + (c16 >> 2) * 16384 + r * 128;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int cc = (c16 & 3) * 2 + q;
    *reinterpret_cast<uint4*>(row + ((cc ^ (r & 7)) << 4)) = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
  }
}

// Zeros rows [first, 128) of a tile that a TMA load has filled, for the tensor core; called by one whole warp.  The rows are those of
// the next document, or padding that may hold anything: what multiplies them is zero, but 0 x NaN is NaN.
template <int PANELS>
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int first) {
  for (int i = first * 8 + static_cast<int>(threadIdx.x & 31); i < 128 * 8; i += 32)
#pragma unroll
    for (int p = 0; p < PANELS; ++p) reinterpret_cast<uint4*>(tile + p * 16384)[i] = make_uint4(0u, 0u, 0u, 0u);
  fence_async_smem();
  __syncwarp();
}

// descriptors over a [128 rows x D] bf16 tile stored as D/64 panels of 16 KB
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t base, int kk) {      // K = columns, k-step of 16 columns
  return umma_smem_desc(base + (kk >> 2) * 16384 + (kk & 3) * 32, 16, 1024);
}
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t base, int kk) {     // K = rows, k-step of 16 rows
  return umma_smem_desc(base + kk * 2048, 16384, 1024);
}

// a warpgroup's share of the registers its CTA was launched with
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// the n lowest of 32 bits, for any n
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

}  // namespace cb
