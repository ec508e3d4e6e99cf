// Rotary positions with the per-head RMS norm of queries and keys in the same pass, and the write of k and v into their
// cache pages.
//
// One CTA per token: its R/2 angles are reduced to a fraction of a turn in 64 bits (position * frequency loses whole radians in
// 32 bits at positions of a million), their sines and cosines in 32 bits go to shared memory and serve every head. A row
// (one head) belongs to a group of lanes, eight channels each: the sum of squares is a shuffle reduction within the group, the
// rotation partner a pair of the same lane (interleaved) or, in the half layout, of the lane R/16 away; a rotated part
// that does not end on that grid goes through shared memory.
#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int TPB = 256;
constexpr int MAX_D = 256;

__device__ __forceinline__ int64_t index_at(const pla_b200_index& x, int64_t i) {
  return x.wide ? static_cast<const int64_t*>(x.data)[i * x.stride] : static_cast<const int32_t*>(x.data)[i * x.stride];
}

template <typename act_t>
__device__ __forceinline__ void unpack(const uint4& raw, float* x) {
  const act_t* e = reinterpret_cast<const act_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}

template <typename act_t>
__device__ __forceinline__ uint4 pack(const float* x) {
  uint4 raw;
  act_t* e = reinterpret_cast<act_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<act_t>(x[i]);
  return raw;
}

template <typename act_t>
__global__ void __launch_bounds__(TPB) rotary_kernel(const pla_b200_rotary_args p, int group) {
  __shared__ float s_cos[MAX_D / 2], s_sin[MAX_D / 2];
  __shared__ float s_w[2][MAX_D];
  __shared__ float s_row[TPB * 8];
  const int tid = threadIdx.x, lane = tid % group, gid = tid / group;
  const int64_t t = blockIdx.x;
  const int e0 = lane * 8, D = p.D, R = p.R, half = p.R / 2;
  const int64_t position = index_at(p.positions, t);
  for (int i = tid; i < half; i += TPB) {
    const double turns = static_cast<double>(position) * p.inv_freq[i] * 0.15915494309189535;   // 1 / (2 pi)
    const float frac = static_cast<float>(turns - rint(turns));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    s_cos[i] = cs * p.factor;
    s_sin[i] = sn * p.factor;
  }
  for (int i = tid; i < 2 * D; i += TPB) {
    const bool second = i >= D;
    const void* w = second ? p.k_weight : p.q_weight;
    if (w != nullptr)
      s_w[second][i - second * D] = load_any(w, second ? p.k_weight_dtype : p.q_weight_dtype, i - second * D) + (p.unit_offset ? 1.0f : 0.0f);
  }
  __syncthreads();
  int64_t block = -1, off = 0;
  if (p.k_cache != nullptr) {
    const int64_t slot = index_at(p.slots, t);
    if (slot >= 0) {
      block = slot / p.block_size;
      off = slot % p.block_size;
      if (block >= p.num_blocks) {
        block = -1;
        if (tid == 0 && p.status != nullptr) atomicOr(p.status, PLA_B200_DEV_BAD_SLOT);
      }
    }
  }
  const int rows = p.Hq + p.Hk, all = rows + (p.k_cache != nullptr ? p.Hk : 0), groups = TPB / group;
  for (int r0 = 0; r0 < all; r0 += groups) {      // uniform over the CTA: the shuffles see every lane
    const int r = r0 + gid;
    const bool live = r < all && e0 < D;
    const int kind = r < p.Hq ? 0 : r < rows ? 1 : 2;
    const int h = kind == 0 ? r : kind == 1 ? r - p.Hq : r - rows;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (live) {
      const act_t* src = kind == 0   ? static_cast<const act_t*>(p.q) + t * p.q_tok_stride + h * p.q_head_stride
                         : kind == 1 ? static_cast<const act_t*>(p.k) + t * p.k_tok_stride + h * p.k_head_stride
                                     : static_cast<const act_t*>(p.v) + t * p.v_tok_stride + h * p.v_head_stride;
      raw = *reinterpret_cast<const uint4*>(src + e0);
    }
    float x[8], y[8];
    unpack<act_t>(raw, x);
    float sq = 0.0f;                              // reduced by every lane: the groups of a warp may be of different kinds
#pragma unroll
    for (int i = 0; i < 8; ++i) sq += x[i] * x[i];
    for (int o = group >> 1; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    if (live && kind < 2 && (kind == 0 ? p.q_weight : p.k_weight) != nullptr) {
      const float inv = rsqrtf(sq / static_cast<float>(D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= inv * s_w[kind][e0 + i];
    }
    float* row = s_row + gid * group * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) row[e0 + i] = x[i];
    __syncwarp();
    if (live && kind < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        if (e >= R) {
          y[i] = x[i];
        } else if (p.interleaved) {
          const int f = e >> 1;
          y[i] = (e & 1) ? x[i] * s_cos[f] + row[e - 1] * s_sin[f] : x[i] * s_cos[f] - row[e + 1] * s_sin[f];
        } else if (e < half) {
          y[i] = x[i] * s_cos[e] - row[e + half] * s_sin[e];
        } else {
          y[i] = x[i] * s_cos[e - half] + row[e - half] * s_sin[e - half];
        }
      }
      const uint4 out = pack<act_t>(y);
      if (kind == 0) {
        *reinterpret_cast<uint4*>(static_cast<act_t*>(p.q_out) + t * p.qo_tok_stride + h * p.qo_head_stride + e0) = out;
      } else {
        if (p.k_out != nullptr)
          *reinterpret_cast<uint4*>(static_cast<act_t*>(p.k_out) + t * p.ko_tok_stride + h * p.ko_head_stride + e0) = out;
        if (block >= 0)
          *reinterpret_cast<uint4*>(static_cast<act_t*>(p.k_cache) + block * p.k_strides.block + off * p.k_strides.token +
                                    h * p.k_strides.head + e0) = out;
      }
    } else if (live && block >= 0) {
      *reinterpret_cast<uint4*>(static_cast<act_t*>(p.v_cache) + block * p.v_strides.block + off * p.v_strides.token +
                                h * p.v_strides.head + e0) = raw;
    }
    __syncwarp();
  }
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
  int group = 1;
  while (group * 8 < a.D) group <<= 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(a.T);
  if (a.act_dtype == PLA_B200_BF16)
    rotary_kernel<__nv_bfloat16><<<grid, TPB, 0, s>>>(a, group);
  else
    rotary_kernel<__half><<<grid, TPB, 0, s>>>(a, group);
  PLA_CUDA_OK(cudaGetLastError());
  return PLA_B200_OK;
}
