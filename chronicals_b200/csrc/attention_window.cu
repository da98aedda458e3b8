// Causal GQA attention of packed documents with a sliding window and sinks, forward, on tcgen05.
//
// A query at position i of its document sees the keys j <= i with i - j < window, and those with j < sinks:
//     O_i = sum_j p_ij V_j,   p_i = softmax over the visible j of scale q_i . k_j
// in one pass over the keys with a running reference maximum and sum.  (Backward: the windowed forms of the kernels in
// attention.cu.)
//
// One CTA: 128 queries of one document and one head.  Its keys are the 128-row blocks of the sinks and those from the first query's
// first key to the diagonal; the blocks between are left out, so the work grows with the window instead of with the document.
// Only blocks that a window's edge or the diagonal cuts test their scores, by one bit mask a row and 32 columns.
//
// Roles: four softmax warps (a thread owns a score row), a warp that issues every MMA, a warp that owns the TMA rings.  P (bf16)
// is the A operand of P V from tensor memory, O accumulates there; the reference maximum is raised only when a block exceeds it
// by 2^8 (probabilities stay below 256, exact enough in fp32 sums and harmless in bf16), which rescales the thread's own O row.
//
// Blocks of 128 keys: an MMA of 64 columns takes 45 - 48 cycles where one of 128 takes 64, and every block costs its waits.
// Two CTAs an SM, 256 tensor-memory columns each:
//   head size 64:  S [0, 128)  O [128, 192)  P [192, 256): the scores go to registers at once, so that the next block's S is computed
//                  beside this block's softmax and P V beside the maximum of the next one's;
//   head size 128: S [0, 128) with P over its first half, O [128, 256): S, softmax and P V one after another, and the second CTA
//                  between them.
// Bound by the softmax's chain: of 3150 cycles a block and warp (head size 64, two warps a scheduler) the exponentials take 1700
// beside the other CTA's (1024 alone, 16 a clock and SM), the rest is loads, maxima and waits that follow one another; leaving
// every MMA out saves 4 %.  Measured, 14 / 2 heads of 64, 32,768 tokens, window 4096: 612 to 635 us by GPU (737 to 710 TFLOP/s of visible
// pairs); 28 / 4 heads of 128, 8192 tokens, window 2048: 215 to 224 us (983 to 943).  On the GPU of the lower figures the form of attention.cu (64 keys a block, two score tiles) took 690 and 221 with
// the same arithmetic, 822 and 232 with one score an instruction.  Tried besides: three and four CTAs an SM with one 64-key score
// tile each 658 and 654 / -, two threads a row 650 / 234, P V in halves with P's half freed early 669 / 218, some exponentials on
// the FMA pipe 618 (one pair in eight) to 690.  The six warps' 168 registers (two CTAs an SM) are too few for the softmax warps: 144
// bytes of spill stores and 384 of loads at head size 64, 84 and 220 at 128.
//
// P is rounded to bf16 (2^-9 on average) because the tensor core takes it so; sums, maxima and O stay in fp32.
#include <algorithm>
#include "attention.cuh"
#include "host_common.h"

namespace cb {

constexpr int WIN_THREADS = 192;                       // 4 softmax warps + the MMA-issuing warp + the TMA warp
constexpr float WIN_RAISE_LOG2 = 8.f;                  // raise the reference maximum only beyond 2^8

template <int D>
struct WinFwd {
  static constexpr bool P_APART = D == 64;
  static constexpr int NS = D == 64 ? 2 : 1;           // depth of the K ring and of the V ring (a stage is free a softmax early)
  static constexpr uint32_t TMEM_COLS = 256, C_O = 128, C_P = P_APART ? 192 : 0;
  static constexpr int TILE = 128 * D * 2;             // Q tile, K or V block: D/64 panels of 16 KB
  static constexpr int OFF_K = TILE;
  static constexpr int OFF_V = TILE * (1 + NS);
  static constexpr int OFF_BAR = TILE * (1 + 2 * NS);
  static constexpr int TOTAL = OFF_BAR + 256 + 1024;
  static_assert(2 * (TOTAL + 1024) <= 228 * 1024, "two CTAs an SM");
};

template <int D>
__global__ void __launch_bounds__(WIN_THREADS, 2)
attn_window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO, const AttnArgs a,
                       int* __restrict__ lo_index) {
  using L = WinFwd<D>;
  constexpr int NS = L::NS;
  constexpr int PANELS = D / 64;
  constexpr uint32_t C_O = L::C_O, C_P = L::C_P;
  constexpr uint32_t IDESC_S = umma_idesc_bf16(128, 128, 0, 0);
  constexpr uint32_t IDESC_PV = umma_idesc_bf16(128, D, 0, 1);

  int start, len, nblk, qb, run, doc;
  int beyond = 0;
  if (!locate_window_tile<false, D == 64>(a, blockIdx.y, start, len, nblk, qb, run, &beyond, &doc)) {
    zero_padding_rows<D>(a, beyond, blockIdx.x);
    return;
  }
  const int h = blockIdx.x;
  const int hkv = h / (a.hq / a.hk);
  // blocks of 128 keys: [0, n_snk) for the sinks, then [n_snk + skip, qb] to the diagonal
  const int from = max(0, qb * 128 - a.window + 1) >> 7;
  const int n_snk = min((a.sinks + 127) >> 7, from);
  const int skip = from - n_snk;
  const int n_kv = qb + 1 - skip;
  const auto block_of = [&](int j) { return j < n_snk ? j : j + skip; };

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::OFF_K;
  uint8_t* sV = smem + L::OFF_V;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);    // [NS]
  uint64_t* v_full = k_full + NS;                                       // [NS]
  uint64_t* k_empty = v_full + NS;                                      // [NS] S of the stage's block complete
  uint64_t* v_empty = k_empty + NS;                                     // [NS] P V of the stage's block complete
  uint64_t* bar_s = v_empty + NS;                                       // S(j) complete
  uint64_t* s_free = bar_s + 1;                                         // 128 arrivals: S(j) is in registers (P apart)
  uint64_t* p_ready = s_free + 1;                                       // 128 arrivals: P(j) written
  uint64_t* bar_o = p_ready + 1;                                        // P V of block j complete (P apart: phase j; else of the last)
  uint64_t* bar_q = bar_o + 1;
  uint64_t* v_clean = bar_q + 1;                                        // the last V block holds nothing of the next document
  uint64_t* o_staged = v_clean + 1;                                     // 128 arrivals: output rows are in shared memory
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_staged + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(k_full + i, 1); mbar_init(v_full + i, 1); mbar_init(k_empty + i, 1); mbar_init(v_empty + i, 1);
    }
    mbar_init(bar_s, 1); mbar_init(s_free, 128); mbar_init(p_ready, 128);
    mbar_init(bar_o, 1); mbar_init(bar_q, 1); mbar_init(v_clean, 1); mbar_init(o_staged, 128);
    mbar_fence_init();
    *abort_flag = a.status[0] != 0 ? 1 : 0;
  }
  __syncthreads();
  if (*abort_flag) return;
  if (warp == 0) { tmem_alloc(tmem_slot, L::TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  // every wait ends in a warp-wide vote, so that the lanes of a warp leave their loop together
  const auto wait_w = [&](uint64_t* bar, uint32_t parity, int code) {
    ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, code) && ok);
    return ok;
  };
  const bool tail = (qb + 1) * 128 > len;              // the last block reaches beyond the document

  if (warp == 5) {
    // ------------------------------------------------------------------ TMA producer: Q once, then the K and V rings
    // (whole warp, warp-uniform control flow, one elected lane issues)
    const int u_start = __shfl_sync(0xffffffffu, start, 0), u_qb = __shfl_sync(0xffffffffu, qb, 0);
    const int u_nkv = __shfl_sync(0xffffffffu, n_kv, 0);
    const int u_snk = __shfl_sync(0xffffffffu, n_snk, 0), u_skip = __shfl_sync(0xffffffffu, skip, 0);
    if (elect_one()) {
      mbar_expect_tx(bar_q, L::TILE);
#pragma unroll
      for (int p = 0; p < PANELS; ++p) tma_load_2d(sQ + p * 16384, &tmQ, bar_q, h * D + p * 64, u_start + u_qb * 128);
    }
    for (int j = 0; j < u_nkv; ++j) {
      const int st = j % NS, row = u_start + (j < u_snk ? j : j + u_skip) * 128;
      if (j >= NS && !wait_w(k_empty + st, ((j / NS) - 1) & 1, CB_ERR_WAIT_EMPTY)) break;
      if (elect_one()) {
        mbar_expect_tx(k_full + st, L::TILE);
#pragma unroll
        for (int p = 0; p < PANELS; ++p) tma_load_2d(sK + st * L::TILE + p * 16384, &tmK, k_full + st, hkv * D + p * 64, row);
      }
      if (j >= NS && !wait_w(v_empty + st, ((j / NS) - 1) & 1, CB_ERR_WAIT_EMPTY)) break;
      if (elect_one()) {
        mbar_expect_tx(v_full + st, L::TILE);
#pragma unroll
        for (int p = 0; p < PANELS; ++p) tma_load_2d(sV + st * L::TILE + p * 16384, &tmV, v_full + st, hkv * D + p * 64, row);
      }
    }
    if (ok && tail) {
      // Rows behind the document come with its last block: those of the next one, or padding that may hold anything.  Their
      // probabilities are zero, and so have the V rows to be: 0 x NaN is NaN.
      const int j = u_nkv - 1, st = j % NS;
      if (wait_w(v_full + st, (j / NS) & 1, CB_ERR_WAIT_FULL)) {
        zero_tile_rows<PANELS>(sV + st * L::TILE, len - qb * 128);
        if (elect_one()) mbar_arrive(v_clean);
      }
    }
    __syncwarp();
  } else if (warp == 4) {
    // ------------------------------------------------------------------ MMA issue
    const int u_nkv = __shfl_sync(0xffffffffu, n_kv, 0);
    const uint32_t u_tmem = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t qa = smem_u32(sQ);
    const auto issue_s = [&](int j) {                  // S(j) = Q K(j)^T
      const int st = j % NS;
      if (!wait_w(k_full + st, (j / NS) & 1, CB_ERR_WAIT_FULL)) return;
      const uint32_t kb = smem_u32(sK + st * L::TILE);
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) umma_f16_ss(u_tmem, desc_kmajor(qa, kk), desc_kmajor(kb, kk), IDESC_S, kk != 0);
        umma_commit(bar_s);
        umma_commit(k_empty + st);
      }
    };
    if (wait_w(bar_q, 0, CB_ERR_WAIT_FULL)) issue_s(0);
    for (int j = 0; j < u_nkv && ok; ++j) {
      const int st = j % NS;
      if (L::P_APART && j + 1 < u_nkv) {                // S(j + 1) beside the softmax of block j
        if (wait_w(s_free, j & 1, CB_ERR_WAIT_TMEM_EMPTY)) issue_s(j + 1);
        if (!ok) break;
      }
      if (!wait_w(v_full + st, (j / NS) & 1, CB_ERR_WAIT_FULL)) break;
      if (tail && j == u_nkv - 1 && !wait_w(v_clean, 0, CB_ERR_WAIT_FULL)) break;
      const uint32_t vb = smem_u32(sV + st * L::TILE);
      if (!wait_w(p_ready, j & 1, CB_ERR_WAIT_TMEM_EMPTY)) break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk)                  // O += P(j) V(j): A = P from tensor memory, 16 bf16 = 8 words a step
          umma_f16_ts(u_tmem + C_O, u_tmem + C_P + kk * 8, desc_mnmajor(vb, kk), IDESC_PV, (j | kk) != 0);
        if (L::P_APART || j == u_nkv - 1) umma_commit(bar_o);
        umma_commit(v_empty + st);
      }
      if (!L::P_APART && ok && j + 1 < u_nkv) issue_s(j + 1);           // over the scores that P(j) leaves: products complete in order
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax: thread r owns score row r
    const int r = tid;
    const uint32_t t_row = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float sl2 = a.scale * LOG2E;
    const float raise = WIN_RAISE_LOG2 / sl2;          // in raw score units
    const int row = qb * 128 + r;                      // within the document
    float m_ref = -INFINITY, l_run = 0.f;

    // One block; MASK: the diagonal or a window's edge cuts it.  False if a wait was given up.
    const auto block = [&](int j, auto mask_c) {
      constexpr bool MASK = decltype(mask_c)::value;
      if (!wait_w(bar_s, j & 1, CB_ERR_WAIT_TMEM_FULL)) return false;
      tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_row + c * 32, s[c]);
      tmem_ld_wait();
      if (L::P_APART) {                                 // the scores are in registers: their columns may take S(j + 1)
        tc_fence_before();
        mbar_arrive(s_free);
      }
      const int k0 = block_of(j) * 128;
      float m[8];                                       // independent chains: the maximum is latency-, not issue-bound
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (MASK) {
          const int at = k0 + c * 32;
          const uint32_t see = low_bits(row + 1 - at) & (~low_bits(row - a.window + 1 - at) | low_bits(a.sinks - at));
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((see >> i & 1u) == 0) s[c][i] = 0xff800000u;            // -inf
        }
#pragma unroll
        for (int i = 0; i < 32; i += 16)
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float x = __uint_as_float(s[c][i + q]), y = __uint_as_float(s[c][i + 8 + q]);
            m[q] = c == 0 && i == 0 ? fmaxf(x, y) : max3(m[q], x, y);
          }
      }
      const float mx = max3(max3(m[0], m[1], m[2]), max3(m[3], m[4], m[5]), fmaxf(m[6], m[7]));
      const bool up = mx > m_ref + raise;               // also true for a row's first visible key (m_ref = -inf)
      // P V of block j - 1 has to be complete before O is rescaled, and (P apart) before its P is overwritten.  (P over S: it came
      // before S(j), which is complete.)
      if (L::P_APART && j > 0) {
        if (!wait_w(bar_o, (j - 1) & 1, CB_ERR_WAIT_TMEM_FULL)) return false;
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, up)) {
        if (j > 0) {                                    // my O row; P V of block j waits for this thread's P
          const float alpha = up ? ex2_approx((m_ref - mx) * sl2) : 1.f;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld_32x16(t_row + C_O + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x16(t_row + C_O + c * 16, o);
          }
          l_run *= alpha;
        }
        if (up) m_ref = mx;
      }
      // a row may have seen no key yet: its scores are all -inf and stand for zeros against any reference
      const float mb = MASK && m_ref == -INFINITY ? 0.f : m_ref * sl2;
      const uint64_t sc = f2_pack(sl2, sl2), nb = f2_pack(-mb, -mb);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t x = f2_fma(f2_pack(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), sc, nb);
          float e0, e1;
          f2_unpack(x, e0, e1);
          e0 = ex2_approx(e0);
          e1 = ex2_approx(e1);
          sum[i & 1] = f2_add(sum[i & 1], f2_pack(e0, e1));
          pk[i] = pack_bf16x2(e0, e1);
        }
        tmem_st_32x16(t_row + C_P + c * 16, pk);
      }
      float r0, r1;
      f2_unpack(f2_add(sum[0], sum[1]), r0, r1);
      l_run += r0 + r1;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_ready);
      return true;
    };
    for (int j = 0; j < n_kv; ++j) {
      // cut by the diagonal, or by the window's edge of the tile's last row
      const bool cut = block_of(j) == qb || block_of(j) * 128 + a.window <= qb * 128 + 127;
      if (!(cut ? block(j, std::true_type()) : block(j, std::false_type()))) break;
    }

    // A block that lies wholly inside its document leaves through shared memory (the Q tile, which the last S product has finished
    // with) and one TMA store per 64-column panel; a document's last, partial block stores row by row, because a TMA box cannot
    // skip the rows that belong to the next document.
    const bool whole = a.o_tma != 0 && (qb + 1) * 128 <= len;          // CTA-uniform
    if (ok && wait_w(bar_o, L::P_APART ? (n_kv - 1) & 1 : 0, CB_ERR_WAIT_TMEM_FULL)) {
      tc_fence_after();
      const bool row_ok = row < len;                    // the TMEM loads below are warp-wide; only the stores are per row
      const float inv = 1.f / l_run;
      const long long t = start + (row_ok ? row : 0);
      CB_DEBUG_CHECK_ST(a.status, t >= 0 && t < a.T, CB_DBG_ATTN_ROW, t);
      uint4* op = reinterpret_cast<uint4*>(a.O + t * a.ldo + static_cast<long long>(h) * D);
      int lo_at = a.o_lo != nullptr && row_ok ? static_cast<int>(t) : -1;
      if (lo_index != nullptr) {
        if (row >= LO_KEYS) lo_at = -1;
        else if (a.T > static_cast<long long>(LO_KEYS) * a.n_docs && row_ok) lo_at = doc * LO_KEYS + row;
        if (h == 0 && row_ok) lo_index[t] = lo_at;
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld_32x32(t_row + C_O + c * 32, o);
        tmem_ld_wait();
        uint32_t w[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) w[q] = pack_bf16x2(__uint_as_float(o[2 * q]) * inv, __uint_as_float(o[2 * q + 1]) * inv);
        if (lo_at >= 0) {
          uint4* lo = reinterpret_cast<uint4*>(a.o_lo + (static_cast<long long>(lo_at) * a.hq + h) * D + c * 32);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = unpack_bf16x2(w[4 * q + i]);
              v[i] = pack_bf16x2(__uint_as_float(o[8 * q + 2 * i]) * inv - f.x, __uint_as_float(o[8 * q + 2 * i + 1]) * inv - f.y);
            }
            lo[q] = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
        if (whole) {
          store_row_chunk32_packed(sQ, r, c, w);
        } else if (row_ok) {
#pragma unroll
          for (int q = 0; q < 4; ++q) op[c * 4 + q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        }
      }
      if (row_ok) a.lse[static_cast<long long>(h) * a.T + t] = m_ref * a.scale + __logf(l_run);
    }
    if (whole) {
      // every softmax thread reports its rows staged (also one that gave up, so that nobody waits without a limit); warp 0 then
      // stores the tile
      fence_async_smem();
      mbar_arrive(o_staged);
      if (warp == 0) {
        wait_w(o_staged, 0, CB_ERR_WAIT_MISC);
        if (ok && elect_one()) {
#pragma unroll
          for (int p = 0; p < PANELS; ++p) tma_store_2d(&tmO, sQ + p * 16384, h * D + p * 64, start + qb * 128);
          tma_store_commit();
          tma_store_wait_all();                         // shared memory is released when the CTA exits
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 0) { tc_fence_after(); tmem_dealloc(tmem, L::TMEM_COLS); }
}

}  // namespace cb

// =========================================================================================== host side
namespace {

template <int D>
int launch(dim3 grid, cudaStream_t s, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo,
           const cb::AttnArgs& a, int* lo_index) {
  constexpr int smem = cb::WinFwd<D>::TOTAL;
  static bool cfg = false;
  if (!cfg) {
    CB_CHECK_CUDA(cudaFuncSetAttribute(cb::attn_window_fwd_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cfg = true;
  }
  cb::attn_window_fwd_kernel<D><<<grid, cb::WIN_THREADS, smem, s>>>(mq, mk, mv, mo, a, lo_index);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace

extern "C" {

// Rows of what the output's rounding left out; the buffer takes lo_rows * hq * D bf16 and T int32
int cb_attn_window_lo_rows(int T, int n_docs, int window) { return cb::lo_rows(T, n_docs, window); }

// q [T, hq, D] (row pitch ldq elements), k / v [T, hk, D]; cu: int32 [n_docs + 1] on the device; window >= 1, sinks >= 0.
// o [T, hq, D] with pitch ldo; lse [hq, T] fp32.  Rows of o before cu[0] and at or beyond cu[n_docs] (padding) are written as zeros,
// their lse entries are left untouched.  o_lo (null: none; size: cb_attn_window_lo_rows): what o's rounding left out
// where few keys are visible, for the backward pass.  D is 64 or 128, hq a multiple of hk.
int cb_attn_window_fwd(const void* q, const void* k, const void* v, void* o, float* lse, const int* cu, int n_docs, int T,
                       int hq, int hk, int D, long long ldq, long long ldk, long long ldv, long long ldo, float scale, int window,
                       int sinks, void* o_lo, int* status, void* stream) {
  if ((D != 64 && D != 128) || hk <= 0 || hq % hk != 0 || T <= 0 || n_docs <= 0 || window < 1 || sinks < 0 ||
      (reinterpret_cast<uintptr_t>(o_lo) & 15) != 0) return -1;
  const long long tiles = (T + 127LL) / 128 + n_docs;
  if (tiles > 65535) return -1;
  CUtensorMap mq, mk, mv, mo;
  int e = cbhost::make_tmap(&mq, q, static_cast<unsigned long long>(hq) * D, T, ldq, 64, 128);
  if (!e) e = cbhost::make_tmap(&mk, k, static_cast<unsigned long long>(hk) * D, T, ldk, 64, 128);
  if (!e) e = cbhost::make_tmap(&mv, v, static_cast<unsigned long long>(hk) * D, T, ldv, 64, 128);
  if (e) return e;
  cb::AttnArgs a = {};
  a.T = T; a.hq = hq; a.hk = hk; a.n_docs = n_docs; a.cu = cu; a.scale = scale;
  a.O = static_cast<cb::bf16*>(o); a.ldo = ldo; a.lse = lse; a.status = status;
  a.o_lo = static_cast<cb::bf16*>(o_lo);
  int* lo_index = o_lo != nullptr && !cb::lo_all(window)
                      ? reinterpret_cast<int*>(a.o_lo + static_cast<long long>(cb::lo_rows(T, n_docs, window)) * hq * D) : nullptr;
  a.window = std::min(window, T); a.sinks = std::min(sinks, T); a.cap = (a.window + 126) / 128 + 1;
  a.o_tma = cbhost::make_tmap(&mo, o, static_cast<unsigned long long>(hq) * D, T, ldo, 64, 128) == 0 ? 1 : 0;
  if (!a.o_tma) mo = mq;                                // O is not TMA-addressable: every block stores row by row
  const dim3 grid(hq, static_cast<unsigned>(tiles));    // x: query head (fastest, the heads of a group share K / V in L2)
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return D == 64 ? launch<64>(grid, s, mq, mk, mv, mo, a, lo_index) : launch<128>(grid, s, mq, mk, mv, mo, a, lo_index);
}

}  // extern "C"
