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
  bf16* o_lo;           // forward, or null: O less its rounding to bf16, rounded itself (for delta); rows: see LO_KEYS
  int cap;              // blocks of 128 that a tile's loop visits at most, sinks apart
  int sink_run;         // backward: query blocks per CTA of a key block that holds sinks
};

// What the rounding of O to bf16 left out is kept for the backward pass where few keys are visible, at most LO_KEYS besides sinks: the
// row sums take O in, and show it in dQ and dK.  Those are all rows of a window that short, else the first LO_KEYS of every document
// (whatever else is in the batch).  Error of the whole gradient against 64 bits, in roundings to bf16, without / with it: window 2
// 1.70 / 1.41, 4 1.60 / 1.45, 8 1.52 / 1.44, 32 1.46 / 1.43; documents of 40 tokens 1.50 / 1.44.
// 9 documents in 8253 tokens, 14 / 2 heads of 64: forward 50.9 -> 51.3 us; the first 128 of a document 52.3, with no gain in the error;
// with a search for the document in the row sums in the place of the index below 11.1 -> 13.1.
constexpr int LO_KEYS = 32;
// The rows lie in o_lo as [lo_rows, hq, D]; unless they are every token's, lo_rows of them in order, int [T] behind them says which of
// them is a token's (-1: none; tokens of no document: anything, so that a reader has to look whether it is one of lo_rows).
__host__ __device__ constexpr bool lo_all(int window) { return window <= LO_KEYS; }
__host__ __device__ constexpr int lo_rows(int T, int n_docs, int window) {
  return lo_all(window) || T <= static_cast<long long>(LO_KEYS) * n_docs ? T : LO_KEYS * n_docs;
}

// The lane that item b falls into where every lane has `mine` of them, and b within that lane; b < the sum of all
__device__ __forceinline__ int lane_of_item(int& b, int mine) {
  const int lane = threadIdx.x & 31;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += v;
  }
  const int src = __ffs(__ballot_sync(0xffffffffu, b < upto)) - 1;
  b -= __shfl_sync(0xffffffffu, upto - mine, src);
  return src;
}

// The tile of a windowed kernel: CTA b's.  Forward, one tile per query block, the last block of a document first; backward, one per
// key block.  Key blocks that hold sinks are seen by every later query of their document: their query blocks are shared out over
// CTAs in runs of a.sink_run, which come first.  blk: the block of the tile, run: of which run (-1: a key block without sinks).
//
// BY_WEIGHT (head size 64): two to 32 documents are handed out by weight, the blocks that a tile's loop visits, at most a.cap: first
// all tiles of full weight, then those of every lower one, of which a document has at most one (14 / 2 heads of 64, 9 documents in 8192 tokens, window 1024,
// backward: 124 us in the order of the documents, 114 so).  More of them go in their order: a search through more lengths than a
// register holds, level by level, takes longer than it saves (40 documents: 74 and 94 us); empty ones behind the 32nd, with which a
// list may have been filled up, do not count.  A single document's tiles are in that
// order already; with heads of 128, whose tiles take more rounds, the order of the documents is the faster one (16 documents, 28 / 4
// heads, window 512: 248 and 260 us).
template <bool BWD, bool BY_WEIGHT>
__device__ __forceinline__ bool locate_window_tile(const AttnArgs& a, int b, int& start, int& len, int& nblk, int& blk, int& run,
                                                   int* beyond = nullptr, int* doc = nullptr) {
  const int lane = threadIdx.x & 31;
  const int with_sinks = BWD ? (a.sinks + 127) >> 7 : 0;
  run = -1;
  for (int d0 = 0; d0 < a.n_docs; d0 += 32) {
    int st = 0, ln = 0;
    if (d0 + lane < a.n_docs) {
      st = min(max(a.cu[d0 + lane], 0), a.T);            // boundaries outside [0, T] or out of order lead to no address outside
      ln = min(max(a.cu[d0 + lane + 1], st), a.T) - st;
    }
    const int nb = (ln + 127) >> 7, ns = min(nb, with_sinks), own = nb - ns;
    const int in_runs = BWD && ns > 0 ? ns * ((nb + a.sink_run - 1) / a.sink_run) : 0;
    const int all = __reduce_add_sync(0xffffffffu, own + in_runs);
    if (b >= all) {
      b -= all;
      continue;
    }
    const auto take = [&](int src) {
      start = __shfl_sync(0xffffffffu, st, src);
      len = __shfl_sync(0xffffffffu, ln, src);
      nblk = (len + 127) >> 7;
      if (doc != nullptr) *doc = d0 + src;
    };
    if (!BY_WEIGHT || a.n_docs == 1 || (a.n_docs > 32 && a.cu[32] < a.cu[a.n_docs])) {
      take(lane_of_item(b, own + in_runs));
      const int n_s = min(nblk, with_sinks), n_runs = n_s > 0 ? n_s * ((nblk + a.sink_run - 1) / a.sink_run) : 0;
      if (b < n_runs) {
        blk = b % n_s;
        run = b / n_s;
      } else {
        blk = BWD ? b - n_runs + n_s : nblk - 1 - b;
      }
      return true;
    }
    if (BWD && with_sinks > 0) {
      const int n = __reduce_add_sync(0xffffffffu, in_runs);
      if (b < n) {
        take(lane_of_item(b, in_runs));
        const int n_s = min(nblk, with_sinks);
        blk = b % n_s;
        run = b / n_s;
        return true;
      }
      b -= n;
    }
    const int full = max(0, own - a.cap + 1), n = __reduce_add_sync(0xffffffffu, full);
    if (b < n) {
      take(lane_of_item(b, full));
      blk = BWD ? min(nblk, with_sinks) + b : nblk - 1 - b;
      return true;
    }
    b -= n;
    for (int w = min(__reduce_max_sync(0xffffffffu, own), a.cap - 1); w >= 1; --w) {
      const unsigned m = __ballot_sync(0xffffffffu, own >= w);
      const int c = __popc(m);
      if (b < c) {
        take(static_cast<int>(__fns(m, 0, b + 1)));
        blk = BWD ? nblk - w : w - 1;
        return true;
      }
      b -= c;
    }
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

// The grid of ceil(T / 128) + n_docs CTAs (per head) holds enough past the last tile for the rows of no document: where n rows lie
// before cu[0] or at and after cu[n_docs] at least ceil(n / 128), since T - n tokens fill at most (T - n + 127 n_docs) / 128 tiles.
// In the forward kernels they write those rows' zeros, 128 rows x D columns each, so the caller need not clear the output first.
template <int D>
__device__ __forceinline__ void zero_padding_rows(const AttnArgs& a, int beyond, int h) {
  const int lead = min(max(a.cu[0], 0), a.T), valid = max(a.cu[a.n_docs], lead);
  const long long row0 = static_cast<long long>(beyond) * 128;
  constexpr int CH = D / 8;                            // 16-byte chunks per row of one head
  for (int i = threadIdx.x; i < 128 * CH; i += blockDim.x) {
    const long long n = row0 + i / CH, t = n < lead ? n : n - lead + valid;
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
