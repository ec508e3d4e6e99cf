// Attention of one new token per request over a paged key/value cache.
//
// One pass over the keys with the running maximum and sum of the softmax: s = scale q.k (kept in units of log2 so that the
// exponential is one instruction), on a new maximum the sum and the output so far are scaled down. One CTA per (request,
// query head); its warps take the tokens in turn, a lane holds every 32nd channel, and the warps' maxima, sums and outputs are joined
// at the end. Scores, sums and outputs are 32-bit; one rounding of the output.
#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int WARPS = 8;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

template <typename act_t, int D>
__global__ void __launch_bounds__(WARPS * 32) paged_decode_kernel(const pla_b200_paged_decode_args p) {
  constexpr int E = D / 32;
  __shared__ float s_m[WARPS], s_l[WARPS], s_o[WARPS][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t b = blockIdx.x / p.Hq;
  const int h = blockIdx.x % p.Hq, hk = h / (p.Hq / p.Hk);
  const act_t* q = static_cast<const act_t*>(p.q) + b * p.q_row_stride + h * p.q_head_stride;
  const act_t* kc = static_cast<const act_t*>(p.k_cache) + hk * p.k_strides.head;
  const act_t* vc = static_cast<const act_t*>(p.v_cache) + hk * p.v_strides.head;
  int64_t len = p.seq_lens[b];
  int32_t bad = 0;
  if (len < 0) bad |= PLA_B200_DEV_BAD_INTERVAL, len = 0;
  const int64_t room = static_cast<int64_t>(p.columns) * p.block_size;
  if (len > room) bad |= PLA_B200_DEV_BAD_INTERVAL, len = room;
  float qs[E], o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    qs[i] = to_f32(q[lane + 32 * i]) * p.scale * LOG2E;
    o[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = warp; j < len; j += WARPS) {
    const int64_t page = p.block_table[b * p.table_row_stride + j / p.block_size];
    if (page < 0 || page >= p.num_blocks) {
      bad |= PLA_B200_DEV_BAD_SLOT;
      continue;
    }
    const int64_t in = j % p.block_size;
    const act_t* k = kc + page * p.k_strides.block + in * p.k_strides.token;
    const act_t* v = vc + page * p.v_strides.block + in * p.v_strides.token;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += qs[i] * to_f32(k[lane + 32 * i]);
    s = warp_sum(s);
    const float top = fmaxf(m, s);
    const float down = top == -INFINITY ? 1.0f : exp2f(m - top), w = top == -INFINITY ? 0.0f : exp2f(s - top);
    m = top;
    l = l * down + w;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = o[i] * down + w * to_f32(v[lane + 32 * i]);
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int i = 0; i < E; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.0f;
  for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w]);
  for (int w = 0; w < WARPS; ++w) sum += s_m[w] == -INFINITY ? 0.0f : s_l[w] * exp2f(s_m[w] - top);
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float x = 0.0f;
    for (int w = 0; w < WARPS; ++w) x += s_m[w] == -INFINITY ? 0.0f : s_o[w][d] * exp2f(s_m[w] - top);
    static_cast<act_t*>(p.out)[(b * p.Hq + h) * D + d] = from_f32<act_t>(sum == 0.0f ? 0.0f : x / sum);
  }
  if (threadIdx.x == 0 && p.lse != nullptr) p.lse[b * p.Hq + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * LN2;
  if (bad != 0 && p.status != nullptr) atomicOr(p.status, bad);
}

template <typename act_t>
void launch(const pla_b200_paged_decode_args& a, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(a.B) * a.Hq);
  switch (a.D) {
    case 64: paged_decode_kernel<act_t, 64><<<grid, WARPS * 32, 0, s>>>(a); break;
    case 96: paged_decode_kernel<act_t, 96><<<grid, WARPS * 32, 0, s>>>(a); break;
    case 128: paged_decode_kernel<act_t, 128><<<grid, WARPS * 32, 0, s>>>(a); break;
    case 192: paged_decode_kernel<act_t, 192><<<grid, WARPS * 32, 0, s>>>(a); break;
    default: paged_decode_kernel<act_t, 256><<<grid, WARPS * 32, 0, s>>>(a); break;
  }
}

bool strides16(const pla_b200_page_strides& s) { return s.block % 8 == 0 && s.token % 8 == 0 && s.head % 8 == 0; }

}  // namespace
}  // namespace pla

extern "C" int64_t pla_b200_paged_decode_workspace_bytes(int32_t B, int32_t Hq, int32_t Hk, int32_t D) {
  if (B < 0 || Hq <= 0 || Hk <= 0 || D <= 0) return -1;
  return 0;
}

extern "C" int pla_b200_paged_decode(const pla_b200_paged_decode_args* args, void* stream) {
  using namespace pla;
  PLA_REQUIRE(args != nullptr, PLA_B200_E_INVALID, "args is NULL");
  pla_b200_paged_decode_args a = *args;
  default_status(a);
  PLA_REQUIRE(a.B >= 0 && a.Hq > 0 && a.Hk > 0 && a.Hq % a.Hk == 0, PLA_B200_E_INVALID,
              "paged decode needs B >= 0 and a positive number of query heads that the key/value heads divide");
  PLA_REQUIRE(a.D == 64 || a.D == 96 || a.D == 128 || a.D == 192 || a.D == 256, PLA_B200_E_UNSUPPORTED,
              "the head size must be 64, 96, 128, 192 or 256");
  PLA_REQUIRE(a.act_dtype == PLA_B200_BF16 || a.act_dtype == PLA_B200_F16, PLA_B200_E_INVALID, "paged decode takes bf16 or fp16");
  if (a.B == 0) return PLA_B200_OK;
  PLA_REQUIRE(static_cast<int64_t>(a.B) * a.Hq <= INT32_MAX, PLA_B200_E_TOO_LARGE, "too many rows");
  PLA_REQUIRE(a.columns >= 0 && a.block_size > 0 && a.num_blocks >= 0, PLA_B200_E_INVALID, "bad block table sizes");
  PLA_REQUIRE(a.q && a.out && a.seq_lens && (a.columns == 0 || a.block_table) && (a.num_blocks == 0 || (a.k_cache && a.v_cache)),
              PLA_B200_E_INVALID, "q, the caches, block_table, seq_lens and out are required");
  PLA_REQUIRE(aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.out) && a.q_row_stride % 8 == 0 &&
                  a.q_head_stride % 8 == 0 && strides16(a.k_strides) && strides16(a.v_strides),
              PLA_B200_E_ALIGN, "q, out and cache rows must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.act_dtype == PLA_B200_BF16) launch<__nv_bfloat16>(a, s);
  else launch<__half>(a, s);
  PLA_CUDA_OK(cudaGetLastError());
  return PLA_B200_OK;
}
