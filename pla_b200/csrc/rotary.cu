// Rotary positions with the per-head RMS norm of queries and keys in the same pass, and the write of k and v into their
// cache pages.
//
// Bound by the bytes of q, k and v, so everything else is arranged around few instructions per byte. A warp takes the rows
// (heads) of one token, or a share of them when there are few tokens; a row belongs to a group of 4, 8 or 16 lanes, and a lane holds
// eight channels of the row's first half and eight of its second. With y = inv x w (inv from the group's sum of squares) and the
// pair's other channel x', the rotated channel is inv (x A + x' B), A = w cos and B = -+ w' sin: weights, sines and cosines are folded
// once per token and side, and a channel costs two multiply-adds. x' is the lane's other half (whole head rotated), the same lane's
// neighbour (interleaved), comes from the lane R/16 away as the raw 16-bit row (up to half the head rotated), or from that lane's cell in
// shared memory (other sizes of the rotated part). Angles: the warp's lanes reduce position * frequency to a fraction of a turn in 64 bits
// (in 32 bits whole radians are lost at positions of a million), take sine and cosine in 32 bits and share them through shared
// memory. Warps are persistent and bring the next rows, of the next token as well, through a ring of 16-byte asynchronous copies,
// each lane into cells of its own.
// On a B200: norm, rotation (64 of 256) and cache write of 32K tokens of 16/2 heads (671 MB) 115 to 120 us, 5.6 to 5.8 TB/s; rotation alone of
// 32,761 tokens, 64 of 128 interleaved, 32/8 heads (671 MB) 118 us, 5.7 TB/s; 1,999 tokens with the norm (41 MB) 12 us; one token 3 us. At 2.6
// instructions per cycle and SM the arithmetic alone takes about 75 us of these; a seventh fewer instructions did not shorten the large
// calls, so what is left is how well reads and writes overlap. Measured and not kept: two channels per instruction (fma.f32x2: the
// register pairs cost more moves than it saves, 61 -> 83 million instructions for the interleaved case), three CTAs per SM (80 registers
// spill, 167 us), angles in 64-bit floating point (the wrapped integers are exact and a few percent faster).
#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int WARPS = 8;
constexpr int MAX_D = 256;
constexpr int RING = 4;          // steps in flight per warp, 1 KB each
constexpr int BLOCKS = 2;        // CTAs per SM

// Where the other channel of a pair is. HALF_LOW: half layout, R a multiple of 16, at most D / 2. HALF_FULL: half layout, R = D, a multiple
// of 16. HALF_QUADS: half layout, R another multiple of 8. PAIRS: interleaved, R a multiple of 8. ANY: everything else.
enum Layout { HALF_LOW = 0, HALF_FULL = 1, HALF_QUADS = 2, PAIRS = 3, ANY = 4 };

// Queries, keys, values of one call: strides in elements, below 2^31.
struct Side {
  const void* in;
  void* out;               // values: none
  const void* weight;
  int in_tok, in_head, out_tok, out_head, heads, first, weight_dtype;     // first: of the steps in front of this side's
};
struct Work {
  Side side[3];
  pla_b200_index positions, slots;
  const double* inv_freq;
  void* cache[3];          // by side; none for queries
  pla_b200_page_strides cache_strides[3];
  int64_t num_blocks;
  Divisor page;
  int T, D, R, steps, interleaved, unit_offset;
  uint32_t split, workers;
  float factor, eps;
  int32_t* status;
};

__device__ __forceinline__ int64_t index_at(const pla_b200_index& x, int64_t i) {
  return x.wide ? static_cast<const int64_t*>(x.data)[i * x.stride] : static_cast<const int32_t*>(x.data)[i * x.stride];
}

template <typename act_t>
__device__ __forceinline__ float2 widen(uint32_t w);
template <>
__device__ __forceinline__ float2 widen<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 widen<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename act_t>
__device__ __forceinline__ void unpack(const uint4& raw, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 two = widen<act_t>((&raw.x)[i]);
    x[2 * i] = two.x, x[2 * i + 1] = two.y;
  }
}

template <typename act_t>
__device__ __forceinline__ uint32_t narrow(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t narrow<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename act_t>
__device__ __forceinline__ uint4 pack(const float* x) {
  return make_uint4(narrow<act_t>(x[0], x[1]), narrow<act_t>(x[2], x[3]), narrow<act_t>(x[4], x[5]), narrow<act_t>(x[6], x[7]));
}

// Eight numbers of shared memory.
__device__ __forceinline__ void read8(float* to, const float* from) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = reinterpret_cast<const float4*>(from)[i];
    to[4 * i] = x.x, to[4 * i + 1] = x.y, to[4 * i + 2] = x.z, to[4 * i + 3] = x.w;
  }
}

// 16 bytes, asynchronously; in groups, of which wait_copies lets `N` be in flight.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float rsqrt_fast(float x) {     // relative error within 2^-22
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 1 / sqrt(mean(x^2) + eps) of a row whose squares leave the range of 32-bit numbers (bf16 rows of magnitude 1e-20 with a tiny eps, or of
// 1e20), as two factors: a power of two that brings the row's largest number, or the root of eps, to about 1, and the rest. The lane's
// pieces of the row are read again, so that ordinary rows keep nothing for it.
template <typename act_t, int GROUP>
__device__ __forceinline__ float2 inverse_scaled(const uint4* low, const uint4* high, float inv_d, float eps) {
  const float root = sqrtf(eps);
  float most = root, sq = 0.0f, x[8];
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    unpack<act_t>(c == 0 ? *low : *high, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[i]));
  }
#pragma unroll
  for (int o = GROUP / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float scale = __int_as_float(max(254 - (__float_as_int(most) >> 23), 1) << 23);       // 2^(127 - exponent); infinity: 2^-126
#pragma unroll 1
  for (int c = 0; c < 2; ++c) {
    unpack<act_t>(c == 0 ? *low : *high, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(x[i] * scale, x[i] * scale, sq);
  }
#pragma unroll
  for (int o = GROUP / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  return make_float2(scale, rsqrt_fast(fmaf(sq, inv_d, root * scale * (root * scale))));
}

template <typename act_t, int GROUP, int LAYOUT>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) rotary_kernel(const __grid_constant__ Work p) {
  constexpr int ROWS = 32 / GROUP;                     // rows per step of a warp
  __shared__ __align__(16) uint4 s_ring[WARPS][RING][2][32];
  __shared__ __align__(16) float s_w[2][MAX_D];
  __shared__ __align__(16) float s_cos[WARPS][MAX_D / 2], s_sin[WARPS][MAX_D / 2];
  __shared__ int64_t s_turn[MAX_D / 2];                // frequencies in turns per position, units of 2^-64
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = p.R, half = R / 2;

  // ---- this warp: steps [begin, end) of ROWS rows each (queries, keys, values) of every stride_t-th token
  const uint32_t share = blockIdx.x * WARPS + warp, part = share % p.split;
  const int stride_t = static_cast<int>(p.workers / p.split), tokens = share < p.workers ? p.T : 0;
  int t = static_cast<int>(share / p.split);
  const int own = lane % GROUP, sub = lane / GROUP, upper = (p.D + 15) / 16 * 8;
  const int e[2] = {own * 8, upper + own * 8};         // the lane's channels: [e[0], e[0] + 8) and [e[1], e[1] + 8)
  const bool on[2] = {e[0] < upper, e[0] < upper && e[1] < p.D};
  const int begin = static_cast<int>(part * static_cast<uint32_t>(p.steps) / p.split);
  const int end = static_cast<int>((part + 1) * static_cast<uint32_t>(p.steps) / p.split);
  auto wide = [](int a, int b) { return static_cast<int64_t>(a) * b; };

  // ---- loads, RING steps ahead
  const uint32_t cells = smem_addr(&s_ring[warp][0][0][lane]);
  int load_t = t, load_s = begin, load_side = begin < p.side[1].first ? 0 : begin < p.side[2].first ? 1 : 2;
  int load_stop = 0, load_h = 0, load_heads = 0;                       // end of the side, row, rows of the side
  int64_t load_step = 0;
  const act_t* load_ptr = nullptr;
  auto enter_side = [&] {
    const Side& x = p.side[load_side];
    load_h = (load_s - x.first) * ROWS + sub;
    load_heads = x.heads;
    load_stop = load_side == 2 ? end : min(end, p.side[load_side + 1].first);
    load_step = wide(ROWS, x.in_head);
    load_ptr = static_cast<const act_t*>(x.in) + e[0] + wide(load_t, x.in_tok) + wide(load_h, x.in_head);
  };
  auto issue = [&](int cell) {
    if (load_t < tokens) {
      const uint32_t to = cells + cell * 1024;
      if (load_h < load_heads) {
        if (on[0]) copy16(to, load_ptr);
        if (on[1]) copy16(to + 512, load_ptr + upper);
      }
      load_h += ROWS;
      load_ptr += load_step;
      if (++load_s == load_stop) {
        if (load_s == end) {
          load_s = begin;
          load_t = load_t < tokens - stride_t ? load_t + stride_t : tokens;
          load_side = begin < p.side[1].first ? 0 : begin < p.side[2].first ? 1 : 2;
        } else {
          do ++load_side; while (load_side < 2 && p.side[load_side + 1].first <= load_s);
        }
        enter_side();                                  // past the last token: an address that is not used
      }
    }
    commit_copies();
  };
#pragma unroll
  for (int i = 0; i < RING; ++i) s_ring[warp][i][0][lane] = s_ring[warp][i][1][lane] = make_uint4(0, 0, 0, 0);   // channels past D stay 0
  enter_side();
#pragma unroll 1
  for (int i = 0; i < RING; ++i) issue(i);

  // ---- what all tokens share
  for (int i = tid; i < half; i += WARPS * 32) {
    const double turns = p.inv_freq[i] * 0.15915494309189535;          // 1 / (2 pi)
    s_turn[i] = __double2ll_rn((turns - rint(turns)) * 18446744073709551616.0);
  }
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const void* w = p.side[side].weight;
    if (w != nullptr)
      for (int i = tid; i < p.D; i += WARPS * 32) s_w[side][i] = load_any(w, p.side[side].weight_dtype, i) + (p.unit_offset ? 1.0f : 0.0f);
  }
  const bool turns_any = begin < p.side[2].first, caches = p.cache[1] != nullptr && end > p.side[1].first;
  int64_t position = 0, slot = -1;
  if (t < tokens) {
    if (turns_any) position = index_at(p.positions, t);
    if (caches) slot = index_at(p.slots, t);
  }
  const int r16 = R / 16;
  const int mate_lane = own < r16 ? lane + r16 : own < 2 * r16 ? lane - r16 : lane;
  const float inv_d = 1.0f / static_cast<float>(p.D);
  float* const cosines = s_cos[warp];
  float* const sines = s_sin[warp];
  int cell = 0;
  __syncthreads();

#pragma unroll 1
  for (; t < tokens; t = t < tokens - stride_t ? t + stride_t : tokens) {
    if (turns_any) {
#pragma unroll 1
      for (int i = lane; i < half; i += 32) {
        // the product wraps at whole turns; its upper half is the fraction in units of 2^-32
        const int frac = static_cast<int>(static_cast<uint64_t>(position) * static_cast<uint64_t>(s_turn[i]) >> 32);
        float sn, cs;
        sincospif(static_cast<float>(frac) * 4.656612873077393e-10f, &sn, &cs);      // 2^-31: half turns
        cosines[i] = cs * p.factor;
        sines[i] = sn * p.factor;
      }
    }
    int64_t block = -1, off = 0;           // where the token's rows go in the caches
    if (slot >= 0) {
      block = slot <= INT32_MAX ? p.page.quotient(static_cast<int>(slot)) : slot / p.page.d;
      off = slot - block * p.page.d;
      if (block >= p.num_blocks) {
        block = -1;
        if (lane == 0 && p.status != nullptr) atomicOr(p.status, PLA_B200_DEV_BAD_SLOT);
      }
    }
    if (t < tokens - stride_t) {           // of the next token
      if (turns_any) position = index_at(p.positions, t + stride_t);
      if (caches) slot = index_at(p.slots, t + stride_t);
    }
    __syncwarp();

#pragma unroll 1
    for (int side = 0; side < 3; ++side) {
      const Side& z = p.side[side];
      const int first = max(begin, z.first), last = side == 2 ? end : min(end, p.side[side + 1].first);
      if (first >= last) continue;
      const int heads = z.heads;
      int h = (first - z.first) * ROWS + sub;
      act_t* cached = nullptr;
      const int64_t cache_step = ROWS * p.cache_strides[side].head;
      if (side > 0 && block >= 0)
        cached = static_cast<act_t*>(p.cache[side]) + block * p.cache_strides[side].block + off * p.cache_strides[side].token +
                 h * p.cache_strides[side].head + e[0];
      if (side == 2) {                     // values: copied
#pragma unroll 1
        for (int s = first; s < last; ++s) {
          wait_copies<RING - 1>();
          if (cached != nullptr) {
            if (h < heads) {
              if (on[0]) *reinterpret_cast<uint4*>(cached) = s_ring[warp][cell][0][lane];
              if (on[1]) *reinterpret_cast<uint4*>(cached + upper) = s_ring[warp][cell][1][lane];
            }
            cached += cache_step;
          }
          issue(cell);
          cell = (cell + 1) & (RING - 1);
          h += ROWS;
        }
        break;
      }
      const bool normed = z.weight != nullptr, dense = z.out != nullptr;
      act_t* out = dense ? static_cast<act_t*>(z.out) + e[0] + wide(t, z.out_tok) + wide(h, z.out_head) : cached;
      const int64_t out_step = dense ? wide(ROWS, z.out_head) : cache_step;
      const bool stored = out != nullptr;              // not: keys of a padding row

      // weights, sines and cosines of the lane's channels
      float A[2][8], B[2][8];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) A[c][i] = 1.0f, B[c][i] = 0.0f;
        if (LAYOUT == HALF_LOW && c == 1) continue;
        if (LAYOUT == ANY) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = e[c] + i;
            if (at < R && on[c]) {
              const bool second = p.interleaved ? (i & 1) : at >= half;
              const int f = p.interleaved ? at >> 1 : second ? at - half : at;
              A[c][i] = cosines[f];
              B[c][i] = second ? sines[f] : -sines[f];
            }
          }
        } else if (LAYOUT == HALF_QUADS) {     // four channels at a time: half is a multiple of four
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const int at = e[c] + i;
            if (at < R && on[c]) {
              const bool second = at >= half;
              const int f = second ? at - half : at;
              const float4 cs = *reinterpret_cast<const float4*>(cosines + f), sn = *reinterpret_cast<const float4*>(sines + f);
              const float sign = second ? 1.0f : -1.0f;
              A[c][i] = cs.x, A[c][i + 1] = cs.y, A[c][i + 2] = cs.z, A[c][i + 3] = cs.w;
              B[c][i] = sign * sn.x, B[c][i + 1] = sign * sn.y, B[c][i + 2] = sign * sn.z, B[c][i + 3] = sign * sn.w;
            }
          }
        } else if (e[c] < R && on[c]) {
          if (LAYOUT == PAIRS) {
            const float4 cs = *reinterpret_cast<const float4*>(cosines + e[c] / 2), sn = *reinterpret_cast<const float4*>(sines + e[c] / 2);
            A[c][0] = A[c][1] = cs.x, A[c][2] = A[c][3] = cs.y, A[c][4] = A[c][5] = cs.z, A[c][6] = A[c][7] = cs.w;
            B[c][1] = sn.x, B[c][3] = sn.y, B[c][5] = sn.z, B[c][7] = sn.w;
#pragma unroll
            for (int i = 0; i < 8; i += 2) B[c][i] = -B[c][i + 1];
          } else {
            const bool second = e[c] >= half;
            const int f = second ? e[c] - half : e[c];
            const float sign = second ? 1.0f : -1.0f;
            read8(A[c], cosines + f);
            read8(B[c], sines + f);
#pragma unroll
            for (int i = 0; i < 8; ++i) B[c][i] *= sign;
          }
        }
      }
      if (normed) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!on[c]) continue;
          float w[8];
          read8(w, s_w[side] + e[c]);
#pragma unroll
          for (int i = 0; i < 8; ++i) A[c][i] *= w[i];
          if (LAYOUT == HALF_LOW && c == 1) continue;
          if (LAYOUT == PAIRS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) B[c][i] *= w[i ^ 1];
          } else if (LAYOUT == ANY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int at = e[c] + i;
              if (at < R) B[c][i] *= s_w[side][p.interleaved ? at ^ 1 : at < half ? at + half : at - half];
            }
          } else if (LAYOUT == HALF_QUADS) {
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const int at = e[c] + i;
              if (at < R) {
                const float4 m = *reinterpret_cast<const float4*>(s_w[side] + (at < half ? at + half : at - half));
                B[c][i] *= m.x, B[c][i + 1] *= m.y, B[c][i + 2] *= m.z, B[c][i + 3] *= m.w;
              }
            }
          } else if (e[c] < R) {
            read8(w, s_w[side] + (e[c] < half ? e[c] + half : e[c] - half));
#pragma unroll
            for (int i = 0; i < 8; ++i) B[c][i] *= w[i];
          }
        }
      }

#pragma unroll 1
      for (int s = first; s < last; ++s) {
        wait_copies<RING - 1>();
        if (LAYOUT == ANY || LAYOUT == HALF_QUADS) __syncwarp();     // the mate's cell may be another lane's copy
        const uint4 raw[2] = {s_ring[warp][cell][0][lane], s_ring[warp][cell][1][lane]};
        float x[2][8], y[2][8];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          unpack<act_t>(raw[c], x[c]);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[c][i] = x[c][i] * A[c][i];
        }
        // the pairs' other channels; channels past R are left out, 0 * infinity must not enter
        if constexpr (LAYOUT == HALF_LOW) {
          uint4 other;
          other.x = __shfl_sync(0xffffffffu, raw[0].x, mate_lane);
          other.y = __shfl_sync(0xffffffffu, raw[0].y, mate_lane);
          other.z = __shfl_sync(0xffffffffu, raw[0].z, mate_lane);
          other.w = __shfl_sync(0xffffffffu, raw[0].w, mate_lane);
          if (e[0] < R) {
            float z[8];
            unpack<act_t>(other, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[0][i] = fmaf(z[i], B[0][i], y[0][i]);
          }
        } else if constexpr (LAYOUT == HALF_FULL) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[0][i] = fmaf(x[1][i], B[0][i], y[0][i]), y[1][i] = fmaf(x[0][i], B[1][i], y[1][i]);
        } else if constexpr (LAYOUT == PAIRS) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (e[c] < R) {
#pragma unroll
              for (int i = 0; i < 8; ++i) y[c][i] = fmaf(x[c][i ^ 1], B[c][i], y[c][i]);
            }
        } else if constexpr (LAYOUT == HALF_QUADS) {
          const act_t* pieces = reinterpret_cast<const act_t*>(&s_ring[warp][cell][0][sub * GROUP]);    // the row's, 256 channels apart
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const int at = e[c] + i, mate = at < half ? at + half : at - half;
              if (on[c] && at < R) {
                const uint2 four = *reinterpret_cast<const uint2*>(pieces + (mate < upper ? mate : mate - upper + 256));
                const float2 lo = widen<act_t>(four.x), hi = widen<act_t>(four.y);
                y[c][i] = fmaf(lo.x, B[c][i], y[c][i]);
                y[c][i + 1] = fmaf(lo.y, B[c][i + 1], y[c][i + 1]);
                y[c][i + 2] = fmaf(hi.x, B[c][i + 2], y[c][i + 2]);
                y[c][i + 3] = fmaf(hi.y, B[c][i + 3], y[c][i + 3]);
              }
            }
          __syncwarp();                                       // the cells are filled again
        } else {
          const act_t* pieces = reinterpret_cast<const act_t*>(&s_ring[warp][cell][0][sub * GROUP]);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int at = e[c] + i, mate = p.interleaved ? at ^ 1 : at < half ? at + half : at - half;
              if (on[c] && at < R) y[c][i] = fmaf(to_f32(pieces[mate < upper ? mate : mate - upper + 256]), B[c][i], y[c][i]);
            }
          __syncwarp();                                       // the cells are filled again
        }
        if (normed) {
          float sq = 0.0f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sq = fmaf(x[i / 8][i % 8], x[i / 8][i % 8], sq);
#pragma unroll
          for (int o = GROUP / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          const float mean = fmaf(sq, inv_d, p.eps);
          float inv = rsqrt_fast(mean);
          if (__any_sync(0xffffffffu, !(mean >= 0x1p-100f && mean < INFINITY))) {
            const float2 two = inverse_scaled<act_t, GROUP>(&s_ring[warp][cell][0][lane], &s_ring[warp][cell][1][lane], inv_d, p.eps);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i / 8][i % 8] *= two.x;
            inv = two.y;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i / 8][i % 8] *= inv;
        }
        if (h < heads && stored) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (!on[c]) continue;
            const uint4 packed = pack<act_t>(y[c]);
            *reinterpret_cast<uint4*>(out + c * upper) = packed;
          }
        }
        issue(cell);
        cell = (cell + 1) & (RING - 1);
        h += ROWS;
        out += out_step;
      }
    }
    __syncwarp();                          // the next token overwrites sines and cosines
  }
  wait_copies<0>();
}

template <typename act_t, int GROUP>
int launch(const pla_b200_rotary_args& a, cudaStream_t stream) {
  constexpr int ROWS = 32 / GROUP;
  const bool cached = a.k_cache != nullptr;
  const int steps_q = (a.Hq + ROWS - 1) / ROWS, steps_k = (a.Hk + ROWS - 1) / ROWS;
  auto i = [](int64_t x) { return static_cast<int>(x); };
  Work w = {};
  w.side[0] = {a.q, a.q_out, a.q_weight, i(a.q_tok_stride), i(a.q_head_stride), i(a.qo_tok_stride), i(a.qo_head_stride), a.Hq, 0, a.q_weight_dtype};
  w.side[1] = {a.k, a.k_out, a.k_weight, i(a.k_tok_stride), i(a.k_head_stride), i(a.ko_tok_stride), i(a.ko_head_stride), a.Hk, steps_q, a.k_weight_dtype};
  w.side[2] = {a.v, nullptr, nullptr, i(a.v_tok_stride), i(a.v_head_stride), 0, 0, cached ? a.Hk : 0, steps_q + steps_k, 0};
  w.positions = a.positions;
  w.inv_freq = a.inv_freq;
  if (cached) {
    w.slots = a.slots;
    w.cache[1] = a.k_cache;
    w.cache[2] = a.v_cache;
    w.cache_strides[1] = a.k_strides;
    w.cache_strides[2] = a.v_strides;
    w.num_blocks = a.num_blocks;
    w.page = Divisor(static_cast<uint32_t>(a.block_size));
  }
  w.T = a.T, w.D = a.D, w.R = a.R, w.interleaved = a.interleaved, w.unit_offset = a.unit_offset;
  w.steps = steps_q + steps_k * (cached ? 2 : 1);
  w.factor = a.factor, w.eps = a.eps, w.status = a.status;
  // A warp per token once that fills the SMs; with fewer tokens their steps are shared out.
  const int64_t full = static_cast<int64_t>(sm_count()) * BLOCKS * WARPS;
  int64_t split = full / a.T;
  split = split < 1 ? 1 : split > w.steps ? w.steps : split;
  const int64_t workers = a.T * split < full ? a.T * split : full / split * split;
  w.split = static_cast<uint32_t>(split);
  w.workers = static_cast<uint32_t>(workers);
  const unsigned grid = static_cast<unsigned>((workers + WARPS - 1) / WARPS);
  if (a.R % 8 != 0) rotary_kernel<act_t, GROUP, ANY><<<grid, WARPS * 32, 0, stream>>>(w);
  else if (a.interleaved) rotary_kernel<act_t, GROUP, PAIRS><<<grid, WARPS * 32, 0, stream>>>(w);
  else if (a.R % 16 == 0 && 2 * a.R <= a.D) rotary_kernel<act_t, GROUP, HALF_LOW><<<grid, WARPS * 32, 0, stream>>>(w);
  else if (a.R % 16 == 0 && a.R == a.D) rotary_kernel<act_t, GROUP, HALF_FULL><<<grid, WARPS * 32, 0, stream>>>(w);
  else rotary_kernel<act_t, GROUP, HALF_QUADS><<<grid, WARPS * 32, 0, stream>>>(w);
  PLA_CUDA_OK(cudaGetLastError());
  return PLA_B200_OK;
}

template <typename act_t>
int launch_for(const pla_b200_rotary_args& a, cudaStream_t s) {
  return a.D <= 64 ? launch<act_t, 4>(a, s) : a.D <= 128 ? launch<act_t, 8>(a, s) : launch<act_t, 16>(a, s);
}

bool strides16(const pla_b200_page_strides& s) { return s.block % 8 == 0 && s.token % 8 == 0 && s.head % 8 == 0; }

}  // namespace
}  // namespace pla

extern "C" int pla_b200_rotary(const pla_b200_rotary_args* args, void* stream) {
  using namespace pla;
  PLA_REQUIRE(args != nullptr, PLA_B200_E_INVALID, "args is NULL");
  pla_b200_rotary_args a = *args;
  default_status(a);
  PLA_REQUIRE(a.T >= 0 && a.Hq >= 0 && a.Hk >= 0, PLA_B200_E_INVALID, "rotary needs T, Hq, Hk >= 0");
  PLA_REQUIRE(a.D > 0 && a.D % 8 == 0 && a.D <= MAX_D, PLA_B200_E_INVALID, "the head size must be a multiple of 8, at most 256");
  PLA_REQUIRE(a.R >= 0 && a.R % 2 == 0 && a.R <= a.D, PLA_B200_E_INVALID, "the rotated part must be even and at most the head size");
  PLA_REQUIRE(a.act_dtype == PLA_B200_BF16 || a.act_dtype == PLA_B200_F16, PLA_B200_E_INVALID, "rotary activations must be bf16 or fp16");
  if (a.T == 0 || a.Hq + a.Hk == 0) return PLA_B200_OK;
  PLA_REQUIRE((a.Hq == 0 || (a.q && a.q_out)) && (a.Hk == 0 || (a.k && (a.k_out || a.k_cache))) && a.positions.data &&
                  (a.inv_freq || a.R == 0),
              PLA_B200_E_INVALID, "q, k, their outputs, positions and inv_freq are required");
  if (a.Hk == 0) a.k_cache = nullptr;
  for (const int64_t stride : {a.q_tok_stride, a.q_head_stride, a.k_tok_stride, a.k_head_stride, a.v_tok_stride, a.v_head_stride, a.qo_tok_stride,
                               a.qo_head_stride, a.ko_tok_stride, a.ko_head_stride})
    PLA_REQUIRE(stride >= 0 && stride <= INT32_MAX, PLA_B200_E_TOO_LARGE, "token and head strides must be below 2^31 elements");
  PLA_REQUIRE(a.Hq < 65536 && a.Hk < 65536, PLA_B200_E_TOO_LARGE, "too many heads");
  if (a.k_cache != nullptr) {
    PLA_REQUIRE(a.k_out == nullptr, PLA_B200_E_INVALID, "keys go either to k_out or to the cache");
    PLA_REQUIRE(a.v_cache && a.v && a.slots.data && a.num_blocks >= 0 && a.block_size > 0, PLA_B200_E_INVALID,
                "a cache needs k_cache, v_cache, v, slots, num_blocks >= 0 and block_size > 0");
    PLA_REQUIRE(aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.v) && strides16(a.k_strides) && strides16(a.v_strides) &&
                    a.v_tok_stride % 8 == 0 && a.v_head_stride % 8 == 0,
                PLA_B200_E_ALIGN, "v and cache rows must be 16-byte aligned");
  }
  PLA_REQUIRE(aligned16(a.q) && aligned16(a.k) && aligned16(a.q_out) && aligned16(a.k_out) && a.q_tok_stride % 8 == 0 &&
                  a.q_head_stride % 8 == 0 && a.k_tok_stride % 8 == 0 && a.k_head_stride % 8 == 0 && a.qo_tok_stride % 8 == 0 &&
                  a.qo_head_stride % 8 == 0 && a.ko_tok_stride % 8 == 0 && a.ko_head_stride % 8 == 0,
              PLA_B200_E_ALIGN, "q, k and output rows must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a.act_dtype == PLA_B200_BF16 ? launch_for<__nv_bfloat16>(a, s) : launch_for<__half>(a, s);
}
