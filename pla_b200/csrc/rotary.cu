// Rotary positions with the per-head RMS norm of queries and keys in the same pass, and the write of k and v into their
// cache pages.
//
// Bound by the bytes of q, k and v, so everything else is arranged around few instructions per byte. A warp takes the rows
// (heads) of one token, or a share of them when there are few tokens; a row belongs to a group of 4, 8 or 16 lanes, and a lane holds
// eight channels of the row's first half and eight of its second. With y = inv x w (inv from the group's sum of squares) and the
// pair's other channel x', the rotated channel is inv (x A + x' B), A = w cos and B = -+ w' sin: weights, sines and cosines are folded
// once per token and side, and a channel costs two multiply-adds, two channels to an instruction. x' is the lane's other half
// (whole head rotated), the same lane's neighbour (interleaved), comes from the lane R/16 away as the raw 16-bit row (up to half the
// head rotated), or from memory again where the rotated part does not fit these. Angles: the warp's lanes reduce position * frequency
// to a fraction of a turn in 64 bits (in 32 bits whole radians are lost at positions of a million), take sine and cosine in 32 bits and
// share them through shared memory. Warps are persistent and bring the next rows, of the next token as well, through a ring of
// 16-byte asynchronous copies into cells that only the copying lane reads.
// MEASURED
#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int WARPS = 8;
constexpr int MAX_D = 256;
constexpr int RING = 4;          // steps in flight per warp, 1 KB each
constexpr int BLOCKS = 2;        // CTAs per SM

// Where the other channel of a pair is: HALF_LOW: R a multiple of 16, at most D / 2; HALF_FULL: R = D, a multiple of 16.
enum Layout { HALF_LOW = 0, HALF_FULL = 1, HALF_ANY = 2, PAIRS = 3 };

__device__ __forceinline__ int64_t index_at(const pla_b200_index& x, int64_t i) {
  return x.wide ? static_cast<const int64_t*>(x.data)[i * x.stride] : static_cast<const int32_t*>(x.data)[i * x.stride];
}

// Two 32-bit numbers per instruction (the pair is one 64-bit register).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return r;
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
__device__ __forceinline__ uint32_t narrow(float2 x);
template <>
__device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(float2 x) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  return r;
}
template <>
__device__ __forceinline__ uint32_t narrow<__half>(float2 x) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  return r;
}

// Eight numbers of shared memory.
__device__ __forceinline__ void read8(float2* to, const float* from) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 x = reinterpret_cast<const float4*>(from)[i];
    to[2 * i] = make_float2(x.x, x.y);
    to[2 * i + 1] = make_float2(x.z, x.w);
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

template <typename act_t, int GROUP, int LAYOUT>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS)
rotary_kernel(const pla_b200_rotary_args p, const uint32_t split, const uint32_t workers, const Divisor page) {
  constexpr int ROWS = 32 / GROUP;                     // rows per step of a warp
  __shared__ __align__(16) uint4 s_ring[WARPS][RING][2][32];
  __shared__ __align__(16) float s_w[2][MAX_D];
  __shared__ __align__(16) float s_cos[WARPS][MAX_D / 2], s_sin[WARPS][MAX_D / 2];
  __shared__ double s_turn[MAX_D / 2];                 // frequencies in turns per position
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int D = p.D, R = p.R, half = R / 2;
  const bool weights = p.q_weight != nullptr || p.k_weight != nullptr;

  // ---- this warp: steps [begin, end) of ROWS rows each (queries, keys, values) of every token of its share
  const uint32_t share = blockIdx.x * WARPS + warp, part = share % split;
  const int64_t stride_t = workers / split;
  int64_t t = share / split;
  const int64_t tokens = share < workers ? p.T : 0;
  const int own = lane % GROUP, sub = lane / GROUP, upper = (D + 15) / 16 * 8;
  const int e[2] = {own * 8, upper + own * 8};         // the lane's channels: [e[0], e[0] + 8) and [e[1], e[1] + 8)
  const bool on[2] = {e[0] < upper, e[0] < upper && e[1] < D};
  const int steps_q = (p.Hq + ROWS - 1) / ROWS, steps_k = (p.Hk + ROWS - 1) / ROWS;
  const int steps = steps_q + steps_k + (p.k_cache != nullptr ? steps_k : 0);
  const int begin = static_cast<int>(part * static_cast<uint32_t>(steps) / split), end = static_cast<int>((part + 1) * static_cast<uint32_t>(steps) / split);

  // ---- loads, RING steps ahead
  const uint32_t cells = smem_addr(&s_ring[warp][0][0][lane]);
  int64_t load_t = t;
  int load_s = begin, load_stop = 0, load_h = 0, load_heads = 0;       // the step that comes next, the end of its side, its row
  const act_t* load_ptr = nullptr;
  int64_t load_stride = 0;
  auto enter_side = [&] {
    const int kind = load_s < steps_q ? 0 : load_s < steps_q + steps_k ? 1 : 2;
    const int start = kind == 0 ? 0 : kind == 1 ? steps_q : steps_q + steps_k;
    load_h = (load_s - start) * ROWS + sub;
    load_heads = kind == 0 ? p.Hq : p.Hk;
    load_stop = min(end, start + (kind == 0 ? steps_q : steps_k));
    const int64_t head = kind == 0 ? p.q_head_stride : kind == 1 ? p.k_head_stride : p.v_head_stride;
    const int64_t tok = kind == 0 ? p.q_tok_stride : kind == 1 ? p.k_tok_stride : p.v_tok_stride;
    load_ptr = static_cast<const act_t*>(kind == 0 ? p.q : kind == 1 ? p.k : p.v) + load_t * tok + load_h * head + e[0];
    load_stride = ROWS * head;
  };
  auto issue = [&](int slot) {
    if (load_t < tokens) {
      const uint32_t to = cells + slot * 1024;
      if (load_h < load_heads) {
        if (on[0]) copy16(to, load_ptr);
        if (on[1]) copy16(to + 512, load_ptr + upper);
      }
      load_h += ROWS;
      load_ptr += load_stride;
      if (++load_s == load_stop) {
        if (load_s == end) load_s = begin, load_t += stride_t;
        enter_side();                                  // past the last token: an address that is not used
      }
    }
    commit_copies();
  };
#pragma unroll
  for (int i = 0; i < RING; ++i) s_ring[warp][i][0][lane] = s_ring[warp][i][1][lane] = make_uint4(0, 0, 0, 0);   // channels past D stay 0
  enter_side();
#pragma unroll
  for (int i = 0; i < RING; ++i) issue(i);

  // ---- what all tokens share
  for (int i = tid; i < half; i += WARPS * 32) s_turn[i] = p.inv_freq[i] * 0.15915494309189535;   // 1 / (2 pi)
  if (weights) {
    for (int i = tid; i < 2 * D; i += WARPS * 32) {
      const int side = i >= D;
      const void* w = side ? p.k_weight : p.q_weight;
      s_w[side][i - side * D] = w == nullptr ? 1.0f : load_any(w, side ? p.k_weight_dtype : p.q_weight_dtype, i - side * D) + (p.unit_offset ? 1.0f : 0.0f);
    }
  }
  const bool turns_any = begin < steps_q + steps_k, caches = p.k_cache != nullptr && end > steps_q;
  int64_t position = 0, slot = -1;
  if (t < tokens) {
    if (turns_any) position = index_at(p.positions, t);
    if (caches) slot = index_at(p.slots, t);
  }
  const int r16 = R / 16;
  const int mate_lane = own < r16 ? lane + r16 : own < 2 * r16 ? lane - r16 : lane;
  const float inv_d = 1.0f / static_cast<float>(D);
  float* const cosines = s_cos[warp];
  float* const sines = s_sin[warp];
  int ring = 0;
  __syncthreads();

#pragma unroll 1
  for (; t < tokens; t += stride_t) {
    if (turns_any) {
      for (int i = lane; i < half; i += 32) {
        const double turns = static_cast<double>(position) * s_turn[i];
        const float frac = static_cast<float>(turns - rint(turns));
        float sn, cs;
        sincospif(2.0f * frac, &sn, &cs);
        cosines[i] = cs * p.factor;
        sines[i] = sn * p.factor;
      }
    }
    int64_t k_at = -1, v_at = -1;          // where the token's rows go in the caches
    if (slot >= 0) {
      const int64_t block = slot <= INT32_MAX ? page.quotient(static_cast<int>(slot)) : slot / p.block_size, off = slot - block * p.block_size;
      if (block < p.num_blocks) {
        k_at = block * p.k_strides.block + off * p.k_strides.token;
        v_at = block * p.v_strides.block + off * p.v_strides.token;
      } else if (lane == 0 && p.status != nullptr) {
        atomicOr(p.status, PLA_B200_DEV_BAD_SLOT);
      }
    }
    if (t + stride_t < tokens) {           // of the next token
      if (turns_any) position = index_at(p.positions, t + stride_t);
      if (caches) slot = index_at(p.slots, t + stride_t);
    }
    __syncwarp();

#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const int first = side == 0 ? begin : max(begin, steps_q), last = side == 0 ? min(end, steps_q) : min(end, steps_q + steps_k);
      if (first >= last) continue;
      const bool normed = (side == 0 ? p.q_weight : p.k_weight) != nullptr, stored = side == 1 && k_at >= 0;
      const int heads = side == 0 ? p.Hq : p.Hk;
      int h = (first - (side == 0 ? 0 : steps_q)) * ROWS + sub;
      const int64_t out_step = ROWS * (side == 0 ? p.qo_head_stride : p.ko_head_stride), cache_step = ROWS * p.k_strides.head;
      act_t* out = static_cast<act_t*>(side == 0 ? p.q_out : p.k_out);
      const bool dense = out != nullptr;
      out += t * (side == 0 ? p.qo_tok_stride : p.ko_tok_stride) + h * (side == 0 ? p.qo_head_stride : p.ko_head_stride) + e[0];
      act_t* cached = static_cast<act_t*>(p.k_cache) + k_at + h * p.k_strides.head + e[0];

      // weights, sines and cosines of the lane's channels
      float2 A[2][4], B[2][4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) A[c][i] = make_float2(1.0f, 1.0f), B[c][i] = make_float2(0.0f, 0.0f);
        if (LAYOUT == HALF_LOW && c == 1) continue;
        if (LAYOUT == HALF_LOW || LAYOUT == HALF_FULL) {
          if (e[c] < R && on[c]) {
            const bool second = e[c] >= half;
            const int f = second ? e[c] - half : e[c];
            const float sign = second ? 1.0f : -1.0f;
            read8(A[c], cosines + f);
            read8(B[c], sines + f);
#pragma unroll
            for (int i = 0; i < 4; ++i) B[c][i] = mul2(B[c][i], make_float2(sign, sign));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = e[c] + i;
            if (at < R && on[c]) {
              const bool second = LAYOUT == PAIRS ? (i & 1) : at >= half;
              const int f = LAYOUT == PAIRS ? at >> 1 : second ? at - half : at;
              reinterpret_cast<float*>(A[c])[i] = cosines[f];
              reinterpret_cast<float*>(B[c])[i] = second ? sines[f] : -sines[f];
            }
          }
        }
      }
      if (normed) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!on[c]) continue;
          float2 w[4];
          read8(w, s_w[side] + e[c]);
#pragma unroll
          for (int i = 0; i < 4; ++i) A[c][i] = mul2(A[c][i], w[i]);
          if (LAYOUT == HALF_LOW && c == 1) continue;
          if (LAYOUT == PAIRS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) B[c][i] = mul2(B[c][i], make_float2(w[i].y, w[i].x));
          } else if (LAYOUT == HALF_ANY) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int at = e[c] + i;
              if (at < R) reinterpret_cast<float*>(B[c])[i] *= s_w[side][at < half ? at + half : at - half];
            }
          } else if (e[c] < R) {
            read8(w, s_w[side] + (e[c] < half ? e[c] + half : e[c] - half));
#pragma unroll
            for (int i = 0; i < 4; ++i) B[c][i] = mul2(B[c][i], w[i]);
          }
        }
      }

#pragma unroll 1
      for (int s = first; s < last; ++s) {
        wait_copies<RING - 1>();
        if (LAYOUT == HALF_ANY) __syncwarp();
        const uint4 raw[2] = {s_ring[warp][ring][0][lane], s_ring[warp][ring][1][lane]};
        float2 x[2][4], y[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[c][i] = widen<act_t>((&raw[c].x)[i]), y[c][i] = mul2(x[c][i], A[c][i]);
        if constexpr (LAYOUT == HALF_LOW) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t other = __shfl_sync(0xffffffffu, (&raw[0].x)[i], mate_lane);
            y[0][i] = fma2(widen<act_t>(e[0] < R ? other : 0), B[0][i], y[0][i]);     // copied channels: 0 * infinity must not enter
          }
        } else if constexpr (LAYOUT == HALF_FULL) {
#pragma unroll
          for (int i = 0; i < 4; ++i) y[0][i] = fma2(x[1][i], B[0][i], y[0][i]), y[1][i] = fma2(x[0][i], B[1][i], y[1][i]);
        } else if constexpr (LAYOUT == PAIRS) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              y[c][i] = fma2(e[c] + 2 * i < R ? make_float2(x[c][i].y, x[c][i].x) : make_float2(0.0f, 0.0f), B[c][i], y[c][i]);
        } else {
          const act_t* pieces = reinterpret_cast<const act_t*>(&s_ring[warp][ring][0][sub * GROUP]);    // the row's, 256 channels apart
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int at = e[c] + i, mate = at < half ? at + half : at - half;
              const float other = on[c] && at < R ? to_f32(pieces[mate < upper ? mate : mate - upper + 256]) : 0.0f;
              reinterpret_cast<float*>(y[c])[i] = fmaf(other, reinterpret_cast<float*>(B[c])[i], reinterpret_cast<float*>(y[c])[i]);
            }
          __syncwarp();                                       // the cells are filled again
        }
        if (normed) {
          float2 q2 = mul2(x[0][0], x[0][0]);
#pragma unroll
          for (int i = 1; i < 8; ++i) q2 = fma2(x[i / 4][i % 4], x[i / 4][i % 4], q2);
          float sq = q2.x + q2.y;
#pragma unroll
          for (int o = GROUP / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
          const float inv = rsqrtf(fmaf(sq, inv_d, p.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i / 4][i % 4] = mul2(y[i / 4][i % 4], make_float2(inv, inv));
        }
        if (h < heads) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (!on[c]) continue;
            const uint4 packed = make_uint4(narrow<act_t>(y[c][0]), narrow<act_t>(y[c][1]), narrow<act_t>(y[c][2]), narrow<act_t>(y[c][3]));
            if (dense) *reinterpret_cast<uint4*>(out + c * upper) = packed;
            if (stored) *reinterpret_cast<uint4*>(cached + c * upper) = packed;
          }
        }
        issue(ring);
        ring = ring + 1 == RING ? 0 : ring + 1;
        h += ROWS;
        out += out_step;
        cached += cache_step;
      }
    }

    // values: copied
#pragma unroll 1
    for (int s = max(begin, steps_q + steps_k); s < end; ++s) {
      wait_copies<RING - 1>();
      const int h = (s - steps_q - steps_k) * ROWS + sub;
      if (h < p.Hk && v_at >= 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (on[c])
            *reinterpret_cast<uint4*>(static_cast<act_t*>(p.v_cache) + v_at + h * p.v_strides.head + e[c]) = s_ring[warp][ring][c][lane];
      }
      issue(ring);
      ring = ring + 1 == RING ? 0 : ring + 1;
    }
    __syncwarp();                          // the next token overwrites sines and cosines
  }
  wait_copies<0>();
}

template <typename act_t, int GROUP>
int launch(const pla_b200_rotary_args& a, cudaStream_t stream) {
  constexpr int ROWS = 32 / GROUP;
  const int64_t steps = (a.Hq + ROWS - 1) / ROWS + static_cast<int64_t>((a.Hk + ROWS - 1) / ROWS) * (a.k_cache != nullptr ? 2 : 1);
  // A warp per token once that fills the SMs; with fewer tokens their steps are shared out.
  const int64_t full = static_cast<int64_t>(sm_count()) * BLOCKS * WARPS;
  int64_t split = full / a.T;
  split = split < 1 ? 1 : split > steps ? steps : split;
  int64_t workers = a.T * split < full ? a.T * split : full / split * split;
  const unsigned grid = static_cast<unsigned>((workers + WARPS - 1) / WARPS);
  const uint32_t n = static_cast<uint32_t>(split), w = static_cast<uint32_t>(workers);
  const Divisor page(a.k_cache != nullptr ? static_cast<uint32_t>(a.block_size) : 1u);
  if (a.interleaved) rotary_kernel<act_t, GROUP, PAIRS><<<grid, WARPS * 32, 0, stream>>>(a, n, w, page);
  else if (a.R % 16 == 0 && 2 * a.R <= a.D) rotary_kernel<act_t, GROUP, HALF_LOW><<<grid, WARPS * 32, 0, stream>>>(a, n, w, page);
  else if (a.R % 16 == 0 && a.R == a.D) rotary_kernel<act_t, GROUP, HALF_FULL><<<grid, WARPS * 32, 0, stream>>>(a, n, w, page);
  else rotary_kernel<act_t, GROUP, HALF_ANY><<<grid, WARPS * 32, 0, stream>>>(a, n, w, page);
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
  if (a.k_cache != nullptr) {
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
