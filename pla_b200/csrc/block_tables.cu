// Block tables and slot maps of a serving step from request lengths: one launch, integers only.
//
// A thread owns one new token. Which request the token belongs to is a search in the offsets, which page it falls in
// a division; the pages a request takes from the free list start at the sum of what the requests before it take, so
// every CTA adds those up for itself (a block scan per 1,024 requests, no exchange between CTAs). The token that opens a page
// (p % block_size == 0) is the one that writes the page's table entry: a page taken by this call always starts with a
// token of this call, because the context's last page is held already.
// The call moves a few bytes per request and 16 per token: what bounds it is the chain of dependent reads (lengths ->
// scan -> free list -> stores) behind one launch (256 requests with one token each 3.3 us, 8 with 40K tokens the same).
#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int TPB = 256;          // threads, and new tokens, per CTA
constexpr int PER = 4;            // requests per thread and scan
constexpr int CHUNK = TPB * PER;

__global__ void __launch_bounds__(TPB) block_tables_kernel(const pla_b200_block_tables_args p, const Divisor page_size) {
  auto pages = [&](int n) { return n > 0 ? page_size.quotient(n - 1) + 1 : 0; };      // that n tokens fill
  __shared__ int32_t s_off[CHUNK + 1];     // offsets of the chunk's requests, none below an earlier one
  __shared__ int32_t s_ctx[CHUNK];         // tokens in the cache; -1: bad metadata, no slots
  __shared__ int64_t s_base[CHUNK];        // first entry of the free list that the request takes
  __shared__ int64_t s_warp[TPB / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int t0 = blockIdx.x * TPB;
  const int t = t0 + tid;
  const bool first_cta = blockIdx.x == 0;  // writes what there is per request
  const int64_t start = p.free_start != nullptr ? max(*p.free_start, 0) : 0;
  const int rows = min(max(p.query_start_loc[p.N], 0), p.tokens);       // the others are padding
  int64_t running = start;
  int64_t slot = -1, pos = 0;
  int32_t bad = 0, highest = 0;            // of the offsets so far
  for (int n0 = 0; n0 < p.N; n0 += CHUNK) {
    const int cnt = min(CHUNK, p.N - n0);
    int32_t off[PER + 1], ctx[PER];
    int need[PER];
    int64_t mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int n = n0 + tid * PER + i;
      off[i] = n <= p.N ? p.query_start_loc[n] : 0;
      ctx[i] = n < p.N ? p.context_lens[n] : 0;
    }
    off[PER] = n0 + tid * PER + PER <= p.N ? p.query_start_loc[n0 + tid * PER + PER] : 0;
    // Offsets that are negative or fall (bad metadata): a request that begins below an earlier offset would share its tokens with another
    // one, and only one of them could enter pages there. It gets none; the search goes by the largest offset up to each request.
    int top[PER + 1];
    bool falls = false;
#pragma unroll
    for (int i = 0; i <= PER; ++i) {
      top[i] = off[i];
      if (n0 + tid * PER + i <= p.N) falls |= off[i] < (i > 0 ? off[i - 1] : highest);
    }
    if (__syncthreads_or(falls)) {
#pragma unroll
      for (int i = 0; i < PER; ++i) s_off[tid * PER + i] = off[i];
      __syncthreads();
      int most = highest;
      for (int j = 0; j < tid * PER; ++j) most = max(most, s_off[j]);
#pragma unroll
      for (int i = 0; i <= PER; ++i) top[i] = most = max(most, off[i]);
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int n = n0 + tid * PER + i;
      need[i] = 0;
      if (n >= p.N) continue;
      const int64_t m = static_cast<int64_t>(off[i + 1]) - off[i];
      if (m < 0 || off[i] < top[i] || ctx[i] < 0 || ctx[i] + m > INT32_MAX) {
        bad |= PLA_B200_DEV_BAD_INTERVAL;
        if (first_cta) p.seq_lens[n] = max(ctx[i], 0);
        s_ctx[tid * PER + i] = -1;
      } else {
        // tokens without a row have no thread that could enter a page for them: they are left out of everything
        const int len = ctx[i] + (min(off[i + 1], rows) - min(off[i], rows)), all = pages(len);
        need[i] = max(min(all, p.columns) - pages(ctx[i]), 0);
        if (off[i + 1] > rows) bad |= PLA_B200_DEV_BAD_INTERVAL;
        if (all > p.columns) bad |= PLA_B200_DEV_TABLE_FULL;
        if (first_cta) p.seq_lens[n] = len;
        s_ctx[tid * PER + i] = ctx[i];
      }
      s_off[tid * PER + i] = top[i];
      if (n + 1 == p.N || tid * PER + i + 1 == CHUNK) s_off[tid * PER + i + 1] = top[i + 1];
      mine += need[i];
    }
    int64_t upto = mine;                   // inclusive scan over the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < TPB / 32; ++w) {
      const int64_t x = s_warp[w];
      if (w < warp) before += x;
      total += x;
    }
    int64_t base = running + before + upto - mine;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s_base[tid * PER + i] = base;
      base += need[i];
    }
    __syncthreads();
    const int32_t lo = s_off[0], hi = s_off[cnt];
    if (t < rows && t >= lo && t < hi) {
      int a = 0, b = cnt;                  // s_off[a] <= t < s_off[b]
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (s_off[mid] <= t) a = mid; else b = mid;
      }
      const int c = s_ctx[a];
      if (c >= 0 && t >= s_off[a] && t < s_off[a + 1]) {
        const int at_token = c + (t - s_off[a]), col = page_size.quotient(at_token), held = pages(c), in_page = at_token - col * p.block_size;
        pos = at_token;
        if (col < p.columns) {
          int32_t* entry = p.block_table + (n0 + a) * p.table_row_stride + col;
          int32_t page = -1;
          if (col < held) {
            page = *entry;
          } else {
            const int64_t at = s_base[a] + col - held;
            if (at < p.free_count) page = p.free_blocks[at]; else bad |= PLA_B200_DEV_NO_BLOCK;
            if (in_page == 0) *entry = page;
          }
          if (page >= 0) slot = static_cast<int64_t>(page) * p.block_size + in_page;
        }
      }
    }
    running += total;
    highest = hi;
    if (!first_cta && lo > t0 + TPB - 1) break;     // the tile's tokens lie behind us
    __syncthreads();                       // the next chunk overwrites the shared arrays
  }
  if (t < p.tokens) {
    p.slot_mapping[t] = slot;
    p.positions[t] = pos;
  }
  if (first_cta && tid == 0)
    *p.free_next = static_cast<int32_t>(min(running, static_cast<int64_t>(p.free_count)));
  if (bad != 0 && p.status != nullptr) atomicOr(p.status, bad);
}

}  // namespace
}  // namespace pla

extern "C" int pla_b200_block_tables(const pla_b200_block_tables_args* args, void* stream) {
  using namespace pla;
  PLA_REQUIRE(args != nullptr, PLA_B200_E_INVALID, "args is NULL");
  pla_b200_block_tables_args a = *args;
  default_status(a);
  PLA_REQUIRE(a.N >= 0 && a.tokens >= 0 && a.columns >= 0 && a.free_count >= 0 && a.block_size > 0, PLA_B200_E_INVALID,
              "block tables need N, tokens, columns, free_count >= 0 and block_size > 0");
  PLA_REQUIRE(a.tokens <= INT32_MAX - TPB && a.N <= INT32_MAX - CHUNK, PLA_B200_E_TOO_LARGE, "too many tokens or requests");
  PLA_REQUIRE(a.query_start_loc && a.free_next && (a.N == 0 || (a.seq_lens && a.context_lens)), PLA_B200_E_INVALID,
              "context_lens, query_start_loc, seq_lens and free_next are required");
  PLA_REQUIRE(a.tokens == 0 || (a.slot_mapping && a.positions), PLA_B200_E_INVALID, "slot_mapping and positions are required");
  PLA_REQUIRE(a.N == 0 || a.columns == 0 || (a.block_table && a.table_row_stride >= a.columns), PLA_B200_E_INVALID,
              "block_table rows must not overlap");
  PLA_REQUIRE(a.free_count == 0 || a.free_blocks, PLA_B200_E_INVALID, "free_blocks is NULL");
  const unsigned grid = static_cast<unsigned>(a.tokens > 0 ? (a.tokens + TPB - 1) / TPB : 1);
  block_tables_kernel<<<grid, TPB, 0, static_cast<cudaStream_t>(stream)>>>(a, Divisor(static_cast<uint32_t>(a.block_size)));
  PLA_CUDA_OK(cudaGetLastError());
  return PLA_B200_OK;
}
