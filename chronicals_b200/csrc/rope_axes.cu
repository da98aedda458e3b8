// Rotary positions with several axes (time, height, width, ...) on the Q and K heads of a packed QKV buffer.
//
// A token has one position per axis and every frequency belongs to one axis: with a(f) the axis of frequency f and
// r = pos[a(f)][t],
//     (x1, x2) -> (x1 c - x2 s, x2 c + x1 s),   c = cos[r][f],  s = sin[r][f]   (s negated for the inverse)
// for the pair f of every Q and K head of token t: f and f + D/2 of a head, or 2f and 2f + 1 (INTERLEAVED).
//
// Bound by memory: Q | K is read and written once.  A warp takes one token, because everything that depends on the
// token alone (its positions, the cos / sin values of its pairs) is then fetched once and kept in registers for all its
// heads: a lane owns 8 pairs of every (32 / lanes-a-head)-th head.  The loads of up to ROPE_BATCH heads are in flight
// before the positions are looked at, so the chain positions -> table -> rotation runs beside them.  28 / 4 heads of 128, 32,768 tokens:
// 85 us, 6.3 TB/s; 14 / 2 heads of 64, 8192 tokens: 8.6 us (of 34 MB, partly from L2).
//
// Beyond the formula the destination may differ from the source (the backward pass leaves the gradient it was given as
// it is): V is then copied along.
#include "common.cuh"

namespace cb {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_BATCH = 4;
constexpr int ROPE_MAX_HALF = 256;       // frequencies of a head (its 32 lanes of 8)

struct RopeAxes {
  uint32_t axis[ROPE_MAX_HALF / 16];     // two bits a frequency
};

template <bool INTERLEAVED>
__global__ void __launch_bounds__(ROPE_THREADS)
rope_axes_kernel(const bf16* src, bf16* dst, const float* __restrict__ cosT, const float* __restrict__ sinT,
                 const long long* __restrict__ pos, long long ld_pos, int n_axes, long long T, int heads, int copied, int D,
                 long long ld_src, long long ld_dst, float sign, long long table_len, const RopeAxes axes) {
  const int half = D / 2, tph = half / 8, hs = 32 / tph;                  // lanes a head, heads a pass
  const int lane = threadIdx.x & 31;
  const long long t = blockIdx.x * static_cast<long long>(ROPE_THREADS / 32) + (threadIdx.x >> 5);
  if (t >= T || lane >= hs * tph) return;
  const int c = lane % tph, h0 = lane / tph;
  // 16 bytes at `a` and `b` of a head: the two halves of 8 pairs, or 16 neighbouring values
  const int a = INTERLEAVED ? c * 16 : c * 8, b = INTERLEAVED ? c * 16 + 8 : half + c * 8;
  const bf16* sp = src + t * ld_src;
  bf16* dp = dst + t * ld_dst;
  uint4 u[ROPE_BATCH][2];
  const auto fetch = [&](int h, int last) {
#pragma unroll
    for (int i = 0; i < ROPE_BATCH; ++i) {
      const int hh = h + i * hs;
      if (hh < last) {
        u[i][0] = *reinterpret_cast<const uint4*>(sp + static_cast<long long>(hh) * D + a);
        u[i][1] = *reinterpret_cast<const uint4*>(sp + static_cast<long long>(hh) * D + b);
      }
    }
  };
  fetch(h0, heads);

  float cs[8], sn[8];
  {
    const uint32_t bits = (axes.axis[c >> 1] >> ((c & 1) * 16)) & 0xffffu;
    const auto row = [&](int ax) {
      const long long p = pos[ax * ld_pos + t];
      return p < 0 ? 0 : (p >= table_len ? table_len - 1 : p);            // never read outside the tables
    };
    if (bits == (bits & 3u) * 0x5555u) {                                  // all eight frequencies belong to one axis
      const long long at = row(bits & 3u) * half + c * 8;
      const float4* cp = reinterpret_cast<const float4*>(cosT + at);
      const float4* np = reinterpret_cast<const float4*>(sinT + at);
      const float4 c0 = cp[0], c1 = cp[1], s0 = np[0], s1 = np[1];
      cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
      sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
    } else {
      long long at[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = i < n_axes ? row(i) * half + c * 8 : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t ax = (bits >> (2 * j)) & 3u;
        const long long p = ax == 0 ? at[0] : ax == 1 ? at[1] : ax == 2 ? at[2] : at[3];
        cs[j] = cosT[p + j];
        sn[j] = sinT[p + j];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sn[j] *= sign;
  }

  for (int h = h0; h < heads; h += ROPE_BATCH * hs) {
    if (h != h0) fetch(h, heads);
#pragma unroll
    for (int i = 0; i < ROPE_BATCH; ++i) {
      const int hh = h + i * hs;
      if (hh < heads) {
        float x[8], y[8], ox[8], oy[8];
        unpack8(u[i][0], x);
        unpack8(u[i][1], y);
        if (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            ox[2 * j] = x[2 * j] * cs[j] - x[2 * j + 1] * sn[j];
            ox[2 * j + 1] = x[2 * j + 1] * cs[j] + x[2 * j] * sn[j];
            oy[2 * j] = y[2 * j] * cs[4 + j] - y[2 * j + 1] * sn[4 + j];
            oy[2 * j + 1] = y[2 * j + 1] * cs[4 + j] + y[2 * j] * sn[4 + j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ox[j] = x[j] * cs[j] - y[j] * sn[j];
            oy[j] = y[j] * cs[j] + x[j] * sn[j];
          }
        }
        *reinterpret_cast<uint4*>(dp + static_cast<long long>(hh) * D + a) = pack8(ox);
        *reinterpret_cast<uint4*>(dp + static_cast<long long>(hh) * D + b) = pack8(oy);
      }
    }
  }
  for (int h = heads + h0; h < heads + copied; h += ROPE_BATCH * hs) {
    fetch(h, heads + copied);
#pragma unroll
    for (int i = 0; i < ROPE_BATCH; ++i) {
      const int hh = h + i * hs;
      if (hh < heads + copied) {
        *reinterpret_cast<uint4*>(dp + static_cast<long long>(hh) * D + a) = u[i][0];
        *reinterpret_cast<uint4*>(dp + static_cast<long long>(hh) * D + b) = u[i][1];
      }
    }
  }
}

}  // namespace cb

extern "C" {

// src / dst: rows of (heads + copied) heads of D values with pitches ld_src / ld_dst, 16-byte aligned; the first `heads` are
// rotated, the `copied` ones behind them copied (0 where dst is src).  pos: int64, axis i at pos + i * ld_pos.  axis: two bits a
// frequency, 16 frequencies a word (host memory).  cos / sin [table_len, D / 2] fp32.
int cb_qk_rope_axes(const void* src, void* dst, const float* cosT, const float* sinT, const long long* pos, long long ld_pos,
                    int n_axes, long long T, int heads, int copied, int D, long long ld_src, long long ld_dst, const unsigned* axis,
                    int interleaved, int inverse, long long table_len, void* stream) {
  if (T < 0 || heads < 0 || copied < 0 || D <= 0 || D % 16 != 0 || D / 2 > cb::ROPE_MAX_HALF || n_axes < 1 || n_axes > 4) return -1;
  if (table_len <= 0 || ld_src % 8 != 0 || ld_dst % 8 != 0) return -1;
  if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(cosT) |
        reinterpret_cast<uintptr_t>(sinT)) & 15) != 0) return -1;
  const long long blocks = (T + cb::ROPE_THREADS / 32 - 1) / (cb::ROPE_THREADS / 32);
  if (blocks > 0x7fffffffLL) return -1;
  if (blocks == 0) return 0;
  cb::RopeAxes ax;
  for (int i = 0; i < cb::ROPE_MAX_HALF / 16; ++i) ax.axis[i] = i * 16 < D / 2 ? axis[i] : 0u;
  const auto kern = interleaved ? cb::rope_axes_kernel<true> : cb::rope_axes_kernel<false>;
  kern<<<static_cast<unsigned>(blocks), cb::ROPE_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const cb::bf16*>(src), static_cast<cb::bf16*>(dst), cosT, sinT, pos, ld_pos, n_axes, T, heads, copied, D, ld_src,
      ld_dst, inverse ? -1.f : 1.f, table_len, ax);
  return static_cast<int>(cudaGetLastError());
}

}  // extern "C"
