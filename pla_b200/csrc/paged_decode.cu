// Attention of one new token per request over a paged key/value cache.
//
// One pass over the keys with the running maximum and sum of the softmax: s = scale q.k in units of log2 (the exponential is one
// instruction), on a new maximum the sum and the output so far are scaled down. The call is bound by the bytes of the cache; with
// eight query heads per key/value head, plain multiply-adds could not keep up with them (16 flops per byte and the conversions), so
// both products run on the matrix unit: S^T = K Q^T with keys as rows, so that groups of up to eight heads waste nothing of an
// m16n8k16 instruction, and O^T = V^T P^T. tcgen05 would want 128 keys by 8 heads in tensor memory and the softmax across its lanes; at
// 24 bytes per cycle and SM the warp-level instruction is busy for a few percent of the time and keeps everything in registers.
//
// Work: units of 64 tokens of one (request, key/value head). Every CTA adds up the lengths itself and takes an equal, consecutive
// range of all units (the lengths are on the device, so the host could not split them), which keeps the SMs equally loaded whatever
// the lengths are and splits a single long request over all of them. A producer warp walks the range and keeps a ring of units in
// shared memory filled; in a unit each of the four other warps takes 16 tokens and keeps its own maxima, sums and output, without a
// barrier between them until the range leaves the (request, head). Where pages hold whole tiles of 16 tokens, a tile is a box of a
// tensor map over the cache, one copy per 64 channels; other page sizes take two producer warps and 16-byte asynchronous copies from
// each row's page (32 requests up to 8K tokens of 8 heads of 128: 93 us in pages of one token, 85 is the floor). Both
// leave the 128-byte swizzle that ldmatrix reads without bank conflicts. Tried before: one bulk copy per row and lane (the lanes' copies
// issue one after another, 480 of 620 instructions per tile of 16 tokens) and every warp loading for itself (290 per tile against 240).
// A part that begins or ends inside a CTA's range goes to the workspace as 32-bit sums, and a second kernel, launched so that it
// waits on the first one's end only, joins the parts in order: no atomics, the same bits every time. Calls with little work go to
// clusters instead, which join their parts through distributed shared memory in the same kernel.
// Device time on a B200, calls captured one after another: 64 requests up to 16K tokens, 16/2 heads of 256 (1.14 GB) 177 us, 6.4 TB/s (192 us
// after half a second of such calls, when the 1,000 W cap has the SMs at 1,815 MHz); one of 128K, 32/8 heads of 128 (0.54 GB) 91 us, 5.9 TB/s; 250 up to 2K,
// 32/4 heads of 64 (0.28 GB) 59 us, 4.8 TB/s; 8 up to 4K, 32/8 of 128 (71 MB) 21 us; one of 777, 16/2 of 128 5.6 us. More than 16 query heads per
// key/value head read the rows once per 16: 16 requests up to 16K, heads of 128, 24 us with 16/1 heads, 48 with 64/1, 11 is the floor of both.
// What is left: about 5 us until a CTA's first rows arrive (lengths, page table and rows are three reads that depend on each other), 10 %
// between the first and the last CTA to finish (SMs get unequal shares of the bandwidth), and 4 us for the join. Handing out the last
// eighth or quarter of the units from a counter evened the CTAs out, but the additional parts cost the join more (91 -> 109 us for 128K);
// shares by tiles and item ends instead of units gained 5 % for 200 requests up to 300 tokens and cost small calls 0.7 us.
// Scores, sums and outputs are 32-bit. The matrix unit takes weights p of the activations' type, so each goes in as two numbers, its rounding and
// what the rounding left, and V is multiplied by both: relative 2^-16 (bf16) or 2^-22 (fp16), far below the output's own rounding.
// fp16 loses small numbers, so its weights are 2^7 (SHIFT) times as large: what is lost of one is at most 2^-32 of the largest. The matrix unit
// cuts every product at about 2^-24 of the number that it adds to, which loses a long tail of small weights behind a large one: the 16
// tokens of a tile are summed from zero, and that sum is added in 32 bits, rounded to nearest. Both together cost the first case 28 %
// more instructions and no time, 3 to 4 % under the power cap, and 9 % in the 64/1 case, whose rows come from L2; packed additions
// (add.f32x2), tiles in groups of two or four and accumulators that begin as constants changed nothing or lost.
#include <cuda.h>

#include <type_traits>

#include "common.cuh"
#include "../../include/pla_b200_attention.h"

namespace pla {
namespace {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;   // of the warps that compute; producers come on top
constexpr int TILE = 16;              // tokens per warp and step
constexpr int UNIT = TILE * WARPS;    // tokens per CTA and step
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float SLACK = 8.0f;         // the running maximum may lag this far (log2) behind: fewer rescalings
// The maximum that a warp keeps is this far (log2) below the scores': weights reach 2^(SHIFT + SLACK), 2^15 of the 65,504 that fp16 holds.
template <typename act_t>
constexpr float SHIFT = 0.0f;
template <>
constexpr float SHIFT<__half> = 7.0f;

// Ring depth, and CTAs per SM that its shared memory leaves room for (of 227 KB): 192 KB of rows in flight per SM.
template <int D>
struct Shape {
  static constexpr int BOXES = (D + 63) / 64;              // 64 channels of a unit's rows, 128 bytes each
  static constexpr int BOX = UNIT * 128;
  static constexpr int ROWS = BOXES * BOX;                 // keys (or values) of a unit
  static constexpr int STAGE = 2 * ROWS;
  static constexpr int CTAS = D > 128 ? 1 : D > 64 ? 2 : 3;
  static constexpr int STAGES = 192 * 1024 / CTAS / STAGE;
  static constexpr int HALF = D / 2;
  static constexpr int OP = HALF + 4;                      // row pitch (floats) of the join buffer
  static constexpr int JOIN = WARPS * 8 * OP * 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + JOIN;   // the ring begins at a multiple of 1,024 bytes
};

struct Plan {              // of one call, the same on host and device
  Divisor page;            // by block_size
  int chunks;              // groups of 8 * NT query heads per key/value head
  int group;               // query heads per key/value head
  int grid;
  float* part_o;           // [2 * grid][8 * NT][D]
  float* part_m;           // [2 * grid][8 * NT]
  float* part_l;
  int4* spans;             // [2 * grid]: the split item that CTA i goes on with (2 i), the one that begins in it (2 i + 1):
                           // {request, item, first CTA, last CTA}, last = -1: none
};

template <typename act_t>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename act_t>
__device__ __forceinline__ float2 widen(uint32_t two);
template <>
__device__ __forceinline__ float2 widen<__nv_bfloat16>(uint32_t two) {
  return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 widen<__half>(uint32_t two) {
  return __half22float2(*reinterpret_cast<const __half2*>(&two));
}

template <typename act_t>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float* c, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma<__half>(float* c, const uint32_t* a, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Box of a cache tensor map: channels from x of one head, TILE tokens of one page, into swizzled shared memory.
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int head, int token, int page, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(x), "r"(head), "r"(token), "r"(page), "r"(smem_addr(bar))
               : "memory");
}
// 16 bytes from global memory; or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
// Arrives on `bar` once the thread's earlier copy16()s have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ int length_of(const pla_b200_paged_decode_args& p, int b, int32_t& bad) {
  const int64_t room = min(static_cast<int64_t>(p.columns) * p.block_size, static_cast<int64_t>(1) << 30);
  const int n = p.seq_lens[b];
  if (n < 0 || n > room) bad |= PLA_B200_DEV_BAD_INTERVAL;
  return n < 0 ? 0 : n > room ? static_cast<int>(room) : n;
}

// A place in the sequence of units: request, its item (key/value head and chunk of its query heads), unit of the item.
struct Place {
  int b, head, chunk, unit, units, len;
};

__device__ __forceinline__ void advance(Place& x, const pla_b200_paged_decode_args& p, int chunks) {
  if (++x.unit < x.units) return;
  x.unit = 0;
  if (++x.chunk < chunks) return;
  x.chunk = 0;
  if (++x.head < p.Hk) return;
  x.head = 0;
  int32_t ignored = 0;
  do {
    if (++x.b >= p.B) {                 // past the end: the caller counts its units and never uses this place
      x.units = 1 << 30;
      x.len = 0;
      return;
    }
    x.len = length_of(p, x.b, ignored);
    x.units = (x.len + UNIT - 1) / UNIT;
  } while (x.units == 0);
}

// i * total / parts without overflow, in 32 bits where that is enough (a 64-bit division is a hundred dependent instructions).
__device__ __forceinline__ int64_t scaled(int64_t i, int64_t total, int64_t parts) {
  const uint64_t x = static_cast<uint64_t>(i * total);
  return ((x | static_cast<uint64_t>(parts)) >> 32) == 0 ? static_cast<uint32_t>(x) / static_cast<uint32_t>(parts)
                                                          : static_cast<int64_t>(x / static_cast<uint64_t>(parts));
}

// Barrier of the warps that compute.
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }

// Thread-block clusters: barrier of all their threads, and a word of another CTA's shared memory.
constexpr int TEAM = 8;
__device__ __forceinline__ void team_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t team_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float team_load(uint32_t addr) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(addr) : "memory");
  return x;
}
__device__ __forceinline__ float4 team_load4(uint32_t addr) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(addr) : "memory");
  return x;
}

// Sixteen query heads at once (NT = 2) with 96, 128 or 256 channels take every register there is, and ptxas spills up to 56 bytes (16 requests
// up to 16K, 32/2 heads of 256: 62 us, 4.7 TB/s).
// Warps that load: rows one by one take two (64 requests up to 8K tokens of 4 heads of 64 67 -> 59 us, of 2 heads of 256 137 -> 98), except
// where the computing warps need the registers (16 query heads of 64, three CTAs per SM: 41.8 us with one, 43.9 with two).
template <int D, int NT, bool BOXED>
constexpr int LOADERS = BOXED || (D == 64 && NT == 2) ? 1 : 2;

// BOXED: pages hold whole tiles, the maps describe the caches. TEAMED: the calls with little work. A cluster of TEAM CTAs takes one
// (request, head), each CTA an equal range of its units, and they join their parts through distributed shared memory: no lengths to add
// up, no workspace, no second kernel.
template <typename act_t, int D, int NT, bool BOXED, bool TEAMED>
__global__ void __launch_bounds__(THREADS + 32 * LOADERS<D, NT, BOXED>, Shape<D>::CTAS)
paged_decode_kernel(const pla_b200_paged_decode_args p, const Plan plan, const __grid_constant__ CUtensorMap k_map,
                    const __grid_constant__ CUtensorMap v_map) {
  using S = Shape<D>;
  constexpr int STAGES = S::STAGES, PRODUCERS = LOADERS<D, NT, BOXED>;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* const smem = raw_smem + ((1024 - (smem_addr(raw_smem) & 1023)) & 1023);
  __shared__ uint64_t s_full[STAGES], s_free[STAGES];
  __shared__ uint16_t s_live[STAGES][WARPS];       // rows of each tile that hold a token
  __shared__ float s_m[WARPS][8 * NT], s_l[WARPS][8 * NT];
  __shared__ const void* s_rows[BOXED ? 1 : 2][BOXED ? 1 : UNIT];
  __shared__ int64_t s_scan[WARPS + PRODUCERS];
  __shared__ int s_place[4];
  __shared__ float s_part_m[8 * NT], s_part_l[8 * NT];    // TEAMED: the CTA's part; its sums take the ring's place at the end
  if (!TEAMED) asm volatile("griddepcontrol.launch_dependents;");
  if (BOXED && threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&k_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&v_map) : "memory");
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int items = p.Hk * plan.chunks;
  int32_t bad = 0;

  // ---- the CTA's range of units
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s_full[i], BOXED ? 1 : 33 * PRODUCERS);       // a producer's lane 0, and every lane's copies
      mbar_init(&s_free[i], WARPS);
    }
    fence_mbar_init();
  }
  // Requests of length zero are nobody's unit.
  auto clear_empty = [&] {
    if (tid >= THREADS) return;
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      int32_t ignored = 0;
      if (length_of(p, b, ignored) != 0) continue;
      act_t* out = static_cast<act_t*>(p.out) + static_cast<int64_t>(b) * p.Hq * D;
      for (int i = tid; i < p.Hq * D / 8; i += THREADS) reinterpret_cast<uint4*>(out)[i] = make_uint4(0, 0, 0, 0);
      if (p.lse != nullptr)
        for (int i = tid; i < p.Hq; i += THREADS) p.lse[static_cast<int64_t>(b) * p.Hq + i] = -INFINITY;
    }
  };
  Place at;
  int item_units = 0;                      // TEAMED: of the cluster's item
  int64_t total = 0, workers = 1, begin, end;
  if constexpr (TEAMED) {
    const int item = blockIdx.x / TEAM, rank = blockIdx.x % TEAM;
    at.b = item / items;
    at.head = (item - at.b * items) / plan.chunks;
    at.chunk = item - at.b * items - at.head * plan.chunks;
    at.len = length_of(p, at.b, bad);
    at.units = (at.len + UNIT - 1) / UNIT;
    item_units = at.units;
    begin = item_units * rank / TEAM;
    end = item_units * (rank + 1) / TEAM;
    at.unit = static_cast<int>(begin);
    if (tid < 8 * NT) s_part_m[tid] = -INFINITY;
    __syncthreads();
  } else {
    const int per = (p.B + THREADS - 1) / THREADS;
    const int lo = min(tid * per, p.B), hi = min(lo + per, p.B);
    int64_t mine = 0;
    for (int b = lo; b < hi; ++b) mine += (length_of(p, b, bad) + UNIT - 1) / UNIT;
    mine *= items;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) s_scan[warp] = upto;
    __syncthreads();
    for (int w = 0; w < WARPS + PRODUCERS; ++w) {
      if (w < warp) upto += s_scan[w];
      total += s_scan[w];
    }
    workers = min(static_cast<int64_t>(gridDim.x), total);
    if (blockIdx.x >= workers) {
      clear_empty();
      if (tid < 2) plan.spans[2 * blockIdx.x + tid] = make_int4(0, 0, 0, -1);
      if (blockIdx.x == 0 && bad != 0 && p.status != nullptr) atomicOr(p.status, bad);
      return;
    }
    begin = scaled(blockIdx.x, total, workers);
    end = scaled(blockIdx.x + 1, total, workers);
    if (begin >= upto - mine && begin < upto) {
      int64_t left = begin - (upto - mine);
      for (int b = lo; b < hi; ++b) {
        int32_t ignored = 0;
        const int64_t units = (length_of(p, b, ignored) + UNIT - 1) / UNIT;
        if (left < units * items) {
          s_place[0] = b;
          const int64_t item = scaled(1, left, units);
          s_place[1] = static_cast<int>(item);
          s_place[2] = static_cast<int>(left - item * units);
          s_place[3] = length_of(p, b, ignored);
          break;
        }
        left -= units * items;
      }
    }
    __syncthreads();
    at.b = s_place[0];
    at.head = s_place[1] / plan.chunks;
    at.chunk = s_place[1] % plan.chunks;
    at.unit = s_place[2];
    at.len = s_place[3];
    at.units = (at.len + UNIT - 1) / UNIT;
  }
  const int count = static_cast<int>(end - begin);

  const uint32_t ring = smem_addr(smem);
  bool timed_out = false;
  if (warp >= WARPS) {
    // ---- producer: token of the lane, that of tile lane % 4 when tiles come as boxes, else of every 32nd of its rows
    auto page_of = [&](int t) -> int {               // -1 past the end
      return t < at.len ? p.block_table[at.b * p.table_row_stride + plan.page.quotient(t)] : -1;
    };
    constexpr int TOKENS = BOXED ? 1 : 2 / PRODUCERS;
    const int first_row = BOXED ? 0 : (warp - WARPS) * TOKENS * 32;       // of the producer's
    auto token = [&](int u) { return at.unit * UNIT + (BOXED ? (lane & 3) * TILE : first_row + u * 32 + lane); };
    int page[TOKENS];
#pragma unroll
    for (int u = 0; u < TOKENS; ++u) page[u] = page_of(token(u));
    for (int i = 0; i < count; ++i) {
      const int stage = i % STAGES, head = at.head;
      int left[TOKENS], in[TOKENS], from[TOKENS];
      bool live[TOKENS];
#pragma unroll
      for (int u = 0; u < TOKENS; ++u) {
        const int t = token(u);
        left[u] = at.len - t;
        in[u] = t - plan.page.quotient(t) * p.block_size;
        from[u] = page[u];
        live[u] = left[u] > 0 && page[u] >= 0 && page[u] < p.num_blocks;
        if (left[u] > 0 && !live[u]) bad |= PLA_B200_DEV_BAD_SLOT;
      }
      if (i + 1 < count) {
        advance(at, p, plan.chunks);
#pragma unroll
        for (int u = 0; u < TOKENS; ++u) page[u] = page_of(token(u));      // used one step later
      }
      // all that can be done before the stage is free has been
      if (i >= STAGES) timed_out = __any_sync(0xffffffffu, !mbar_wait(&s_free[stage], (i / STAGES - 1) & 1));
      if (timed_out) break;
      const uint32_t to = ring + stage * S::STAGE;
      uint64_t* const bar = &s_full[stage];
      if constexpr (BOXED) {
        if (lane < WARPS) s_live[stage][lane] = live[0] ? 0xffffu >> (TILE - min(left[0], TILE)) : 0;
        const uint32_t tiles = __ballot_sync(0xffffffffu, live[0]) & 0xfu;
        __syncwarp();
        if (lane == 0) mbar_expect_tx(bar, __popc(tiles) * (2 * S::BOXES * TILE * 128));
        __syncwarp();
        if (lane < WARPS && live[0]) {
          const uint32_t row = to + lane * (TILE * 128);
#pragma unroll
          for (int c = 0; c < S::BOXES; ++c) load_box(row + c * S::BOX, &k_map, c * 64, head, in[0], from[0], bar);
#pragma unroll
          for (int c = 0; c < S::BOXES; ++c) load_box(row + S::ROWS + c * S::BOX, &v_map, c * 64, head, in[0], from[0], bar);
        }
      } else {
        // Row addresses go through shared memory; then a lane keeps one 16-byte column and takes every RPS-th row of it.
        constexpr int COLUMNS = D / 8, RPS = 32 / COLUMNS;                // lanes past RPS * COLUMNS have none (D = 96, 192)
        uint32_t rows[TOKENS];
#pragma unroll
        for (int u = 0; u < TOKENS; ++u) {
          rows[u] = __ballot_sync(0xffffffffu, live[u]);
          const act_t *k_row = static_cast<const act_t*>(p.q), *v_row = k_row;    // a valid address for rows that are not read
          if (live[u]) {
            k_row = static_cast<const act_t*>(p.k_cache) + from[u] * p.k_strides.block + in[u] * p.k_strides.token + head * p.k_strides.head;
            v_row = static_cast<const act_t*>(p.v_cache) + from[u] * p.v_strides.block + in[u] * p.v_strides.token + head * p.v_strides.head;
          }
          s_rows[0][first_row + u * 32 + lane] = k_row;
          s_rows[1][first_row + u * 32 + lane] = v_row;
        }
        if (lane < 2 * TOKENS) s_live[stage][first_row / TILE + lane] = static_cast<uint16_t>(rows[lane >> 1] >> ((lane & 1) * 16));
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
        const int c = lane % COLUMNS, sub = lane / COLUMNS;
        if (sub < RPS) {
          // row r of the column sits at r * 128 + (((c & 7) ^ (r & 7)) << 4); r = sub + a multiple of RPS, whose bits are apart
          const uint32_t dst = to + (c >> 3) * S::BOX + sub * 128, swizzle = ((c & 7) ^ sub) << 4;
          constexpr int AHEAD = 8;                                        // addresses read before their copies are issued
          auto bring = [&](auto all) {
#pragma unroll 1
            for (int r0 = first_row; r0 < first_row + TOKENS * 32; r0 += AHEAD * RPS) {
              const act_t* at_row[2][AHEAD];
#pragma unroll
              for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int side = 0; side < 2; ++side) at_row[side][u] = static_cast<const act_t*>(s_rows[side][r0 + u * RPS + sub]) + c * 8;
              const uint32_t here = rows[TOKENS - 1 && (r0 & 32)] >> ((r0 & 31) + sub);   // AHEAD * RPS divides 32
#pragma unroll
              for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                  const uint32_t at = dst + side * S::ROWS + (r0 + u * RPS) * 128 + (swizzle ^ (((r0 + u * RPS) & 7) << 4));
                  if constexpr (all.value) copy16(at, at_row[side][u]);
                  else copy16(at, at_row[side][u], (here >> (u * RPS)) & 1);
                }
            }
          };
          if ((rows[0] & rows[TOKENS - 1]) == 0xffffffffu) bring(std::true_type{});
          else bring(std::false_type{});
        }
        copies_arrive(bar);
        __syncwarp();                                                     // s_rows is written again
      }
    }
    if (timed_out) bad |= PLA_B200_DEV_WAIT_TIMEOUT;
    if (bad != 0 && p.status != nullptr) atomicOr(p.status, bad);
    if constexpr (TEAMED) {
      __syncwarp();
      team_barrier();
      team_barrier();
    }
    return;
  }
  if (!TEAMED) clear_empty();

  // ---- the lane's part of the running state: heads 2 (lane % 4) and the next of each group of eight
  float m[NT][2], l[NT][2], o[D / 16][NT][4];
  uint32_t qf[D / 16][NT][2];
  const float to_log2 = p.scale * LOG2E;
  auto load_q = [&](const Place& x) {
    const int head = x.head * plan.group + x.chunk * 8 * NT, heads = min(8 * NT, plan.group - x.chunk * 8 * NT);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int h = n * 8 + lane / 4;
      const act_t* q = static_cast<const act_t*>(p.q) + x.b * p.q_row_stride + (head + h) * p.q_head_stride + (lane % 4) * 2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[kk][n][0] = h < heads ? *reinterpret_cast<const uint32_t*>(q + kk * 16) : 0;
        qf[kk][n][1] = h < heads ? *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8) : 0;
      }
    }
  };
  auto clear = [&] {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[kk][n][i] = 0.0f;
    }
  };

  // Joins the four warps' parts of the item that ends here (or leaves the range) and stores them: as output, or as a part.
  // A NaN score leaves the maximum where it is and makes the sum NaN: what has no weight is known by its sum, not by its maximum.
  auto flush = [&](const Place& x, bool whole, int slot) {
    const int head = x.head * plan.group + x.chunk * 8 * NT, heads = min(8 * NT, plan.group - x.chunk * 8 * NT);
    const int64_t first_row = static_cast<int64_t>(x.b) * p.Hq + head, first_part = static_cast<int64_t>(slot) * 8 * NT;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], s);
        if (lane < 4) {
          s_m[warp][n * 8 + lane * 2 + i] = m[n][i];
          s_l[warp][n * 8 + lane * 2 + i] = l[n][i];
        }
      }
    compute_barrier();
    float* join = reinterpret_cast<float*>(smem + STAGES * S::STAGE);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float down[2];                       // what the lane's two heads are multiplied by
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int h = n * 8 + (lane % 4) * 2 + i;
        float top = -INFINITY, weight = 0.0f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, s_m[w][h]);
        const float base = top == -INFINITY ? 0.0f : top;       // exp2(-inf - base) = 0
#pragma unroll
        for (int w = 0; w < WARPS; ++w) weight += s_l[w][h] * fast_exp2(s_m[w][h] - base);
        down[i] = fast_exp2(m[n][i] - base);
        if (whole) down[i] = weight == 0.0f ? 0.0f : down[i] / weight;
        if (warp == 0 && lane < 4 && h < heads) {
          if (!whole) {
            (TEAMED ? s_part_m : plan.part_m + first_part)[h] = top;
            (TEAMED ? s_part_l : plan.part_l + first_part)[h] = weight;
          } else if (p.lse != nullptr) {
            p.lse[first_row + h] = weight == 0.0f ? -INFINITY : (top + log2f(weight)) * LN2;
          }
        }
      }
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        float* mine = join + warp * 8 * S::OP;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          const float* c = o[part * (D / 32) + kk][n];
          float* to = mine + (lane % 4) * 2 * S::OP + kk * 16 + lane / 4;
          to[0] = c[0] * down[0];
          to[S::OP] = c[1] * down[1];
          to[8] = c[2] * down[0];
          to[S::OP + 8] = c[3] * down[1];
        }
        compute_barrier();
#pragma unroll
        for (int i = tid; i < 2 * S::HALF; i += THREADS) {       // four channels of a head
          const int h = i / (S::HALF / 4), d = i % (S::HALF / 4) * 4, hh = n * 8 + h;
          if (hh >= heads) continue;
          float4 sum = *reinterpret_cast<const float4*>(join + h * S::OP + d);
#pragma unroll
          for (int w = 1; w < WARPS; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(join + (w * 8 + h) * S::OP + d);
            sum.x += y.x, sum.y += y.y, sum.z += y.z, sum.w += y.w;
          }
          if (whole)
            *reinterpret_cast<uint2*>(static_cast<act_t*>(p.out) + (first_row + hh) * D + part * S::HALF + d) =
                make_uint2(pack2<act_t>(sum.x, sum.y), pack2<act_t>(sum.z, sum.w));
          else
            *reinterpret_cast<float4*>((TEAMED ? reinterpret_cast<float*>(smem) : plan.part_o + first_part * D) + hh * D + part * S::HALF + d) = sum;
        }
        if (part == 0 || n + 1 < NT) compute_barrier();            // the buffer is written again
      }
    }
  };

  // The CTA that holds unit u.
  auto holder = [&](int64_t u) { return static_cast<int>(scaled(1, (u + 1) * workers - 1, total)); };
  int first_unit = at.unit;
  int4 goes_on = make_int4(0, 0, 0, -1), begins = make_int4(0, 0, 0, -1);
  if (!TEAMED && first_unit > 0) goes_on = make_int4(at.b, at.head * plan.chunks + at.chunk, holder(begin - first_unit), holder(begin + at.units - 1 - first_unit));
  clear();
  if (count > 0) load_q(at);
  int late = 0;
  for (int i = 0; i < count; ++i) {
    const int stage = i % STAGES;
    if (!timed_out && __any_sync(0xffffffffu, !mbar_wait(&s_full[stage], (i / STAGES) & 1))) {
      timed_out = true;
      late = i;
    }
    const uint32_t live = s_live[stage][warp];
    const uint32_t k_rows = ring + stage * S::STAGE + warp * (TILE * 128), v_rows = k_rows + S::ROWS;
    if (live != 0 && !timed_out) {
      if (BOXED && live != 0xffffu) {      // rows of the page past the request's end: p = 0 there, but 0 * garbage need not be 0
        for (int k = lane; k < S::BOXES * TILE * 8; k += 32)
          if (!((live >> ((k >> 3) & 15)) & 1))
            *reinterpret_cast<uint4*>(smem + (v_rows - ring) + (k >> 7) * S::BOX + (k & 127) * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
        __syncwarp();
      }
      // scores of 16 tokens: lane holds tokens lane / 4 and + 8, heads 2 (lane % 4) and + 1
      float s[NT][2][4] = {};
      const uint32_t ka = k_rows + ((lane & 7) + ((lane >> 3) & 1) * 8) * 128;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[4];
        ldmatrix4(a, ka + (kk / 4) * S::BOX + ((((kk % 4) * 2 + (lane >> 4)) ^ (lane & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) mma<act_t>(s[n][kk & 1], a, qf[kk][n]);
      }
      uint32_t pf[NT][2], rest[NT][2];       // weights, and what their rounding left
      float next[NT][2];
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* c = s[n][0];
#pragma unroll
        for (int e = 0; e < 4; ++e) c[e] = (c[e] + s[n][1][e]) * to_log2;
        if (live != 0xffffu) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!((live >> (lane / 4 + (e < 2 ? 0 : 8))) & 1)) c[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(c[e], c[e + 2]);
#pragma unroll
          for (int b = 4; b < 32; b <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
          next[n][e] = x - SHIFT<act_t>;
          grow |= next[n][e] > m[n][e] + SLACK;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float down[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float top = fmaxf(m[n][e], next[n][e]);
            down[e] = m[n][e] == -INFINITY ? 0.0f : fast_exp2(m[n][e] - top);
            m[n][e] = top;
            l[n][e] *= down[e];
          }
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            o[kk][n][0] *= down[0];
            o[kk][n][1] *= down[1];
            o[kk][n][2] *= down[0];
            o[kk][n][3] *= down[1];
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* c = s[n][0];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float top = m[n][e & 1];
          c[e] = fast_exp2(c[e] - (top == -INFINITY ? 0.0f : top));
          l[n][e & 1] += c[e];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t two = pack2<act_t>(c[2 * h], c[2 * h + 1]);
          const float2 kept = widen<act_t>(two);
          pf[n][h] = transpose8x8(two);
          rest[n][h] = transpose8x8(pack2<act_t>(c[2 * h] - kept.x, c[2 * h + 1] - kept.y));
        }
      }
      const uint32_t va = v_rows + ((lane & 7) + (lane >> 4) * 8) * 128;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        uint32_t a[4];
        ldmatrix4_trans(a, va + (kk / 4) * S::BOX + ((((kk % 4) * 2 + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float sum[4] = {};
          mma<act_t>(sum, a, pf[n]);
          mma<act_t>(sum, a, rest[n]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[kk][n][e] += sum[e];
        }
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&s_free[stage]);
    if (at.unit + 1 == at.units || i + 1 == count) {
      const bool whole = !TEAMED && first_unit == 0 && at.unit + 1 == at.units;
      const int slot = TEAMED ? 0 : 2 * blockIdx.x + (first_unit == 0 ? 1 : 0);
      if (!TEAMED && first_unit == 0 && !whole)
        begins = make_int4(at.b, at.head * plan.chunks + at.chunk, blockIdx.x, holder(end + at.units - 2 - at.unit));
      const Place done = at;
      advance(at, p, plan.chunks);
      if (i + 1 < count) load_q(at);          // arrives while the parts are joined
      flush(done, whole, slot);
      clear();
      first_unit = 0;
    } else {
      ++at.unit;
    }
  }
  if (timed_out) {               // a copy never came: say so, and give those in flight time to land before the CTA's memory goes
    bad |= PLA_B200_DEV_WAIT_TIMEOUT;
    for (int i = late; i < min(late + STAGES, count); ++i) mbar_wait(&s_full[i % STAGES], (i / STAGES) & 1);
  }
  if (bad != 0 && p.status != nullptr) atomicOr(p.status, bad);
  if constexpr (TEAMED) {
    __syncwarp();
    team_barrier();                        // all parts are in place
    const int item = blockIdx.x / TEAM, rank = blockIdx.x % TEAM, b = item / items;
    const int head = (item - b * items) / plan.chunks, chunk = item - b * items - head * plan.chunks;
    const int heads = min(8 * NT, plan.group - chunk * 8 * NT), each = (heads * (D / 4) + TEAM - 1) / TEAM;
    const int i = rank * each + tid, h = i / (D / 4), d = i % (D / 4) * 4;       // four channels of a head
    if (tid < each && h < heads) {
      float part_m[TEAM], top = -INFINITY, weight = 0.0f;
      float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int r = 0; r < TEAM; ++r) part_m[r] = team_load(team_addr(smem_addr(&s_part_m[h]), r));
#pragma unroll
      for (int r = 0; r < TEAM; ++r) top = fmaxf(top, part_m[r]);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int r = 0; r < TEAM; ++r) {
        if (item_units * r / TEAM == item_units * (r + 1) / TEAM) continue;       // had no units and stored nothing
        const float f = fast_exp2(part_m[r] - base);
        const float4 x = team_load4(team_addr(ring + (h * D + d) * 4, r));
        weight += team_load(team_addr(smem_addr(&s_part_l[h]), r)) * f;
        sum.x += x.x * f, sum.y += x.y * f, sum.z += x.z * f, sum.w += x.w * f;
      }
      const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
      const int64_t out = static_cast<int64_t>(b) * p.Hq + head * plan.group + chunk * 8 * NT + h;
      *reinterpret_cast<uint2*>(static_cast<act_t*>(p.out) + out * D + d) =
          make_uint2(pack2<act_t>(sum.x * inv, sum.y * inv), pack2<act_t>(sum.z * inv, sum.w * inv));
      if (d == 0 && p.lse != nullptr) p.lse[out] = weight == 0.0f ? -INFINITY : (top + log2f(weight)) * LN2;
    }
    __syncwarp();
    team_barrier();                        // nobody reads this CTA's shared memory any more
  } else if (tid == 0) {
    plan.spans[2 * blockIdx.x] = goes_on;
    plan.spans[2 * blockIdx.x + 1] = begins;
  }
}

// Joins the parts of every item that lies in several CTAs' ranges; CTA 2 i does the item that main CTA i goes on with, CTA 2 i + 1 the
// one that begins there. The CTAs of an item share its heads: the j-th of n takes heads j, j + n, ...; a head's parts are spread
// over the warps, a lane holds four channels of every 128. Small on purpose: its instructions come from memory, not from a warm cache.
constexpr int JOIN_WARPS = 8, AT_ONCE = 4;

template <typename act_t, int D, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const pla_b200_paged_decode_args p, const Plan plan) {
  constexpr int C = (D + 127) / 128;
  __shared__ float s_m[JOIN_WARPS], s_l[JOIN_WARPS];
  __shared__ float4 s_o[JOIN_WARPS][D / 4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 span = plan.spans[blockIdx.x];
  if (span.w < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = span.y % plan.chunks, heads = min(8 * NT, plan.group - chunk * 8 * NT);
  const int parts = span.w - span.z + 1, rank = blockIdx.x / 2 - span.z;
  const int mine = rank < heads ? (heads - rank + parts - 1) / parts : 0;      // heads of this CTA: at most 8 of 16, as parts > 1
  if (mine == 0) return;
  int slices = JOIN_WARPS;                                                     // warps per head
  while (slices * mine > JOIN_WARPS) slices >>= 1;
  const int slot = warp / slices, slice = warp % slices, h = rank + slot * parts;
  float top = -INFINITY, weight = 0.0f;
  float4 sum[C] = {};
  if (slot < mine) {
    for (int j0 = slice; j0 < parts; j0 += AT_ONCE * slices) {
      float m[AT_ONCE], l[AT_ONCE], next = top;
      float4 x[AT_ONCE][C];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int j = j0 + u * slices;
        const bool on = j < parts;
        const int64_t at = static_cast<int64_t>(2 * (span.z + j) + (j == 0 ? 1 : 0)) * 8 * NT + h;
        m[u] = on ? plan.part_m[at] : -INFINITY;
        l[u] = on ? plan.part_l[at] : 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
          x[u][c] = on && c * 32 + lane < D / 4 ? reinterpret_cast<const float4*>(plan.part_o + at * D)[c * 32 + lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) next = fmaxf(next, m[u]);
      const float base = next == -INFINITY ? 0.0f : next;       // exp2(-inf - base) = 0
      const float down = fast_exp2(top - base);
      top = next;
      weight *= down;
#pragma unroll
      for (int c = 0; c < C; ++c) sum[c].x *= down, sum[c].y *= down, sum[c].z *= down, sum[c].w *= down;
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const float f = fast_exp2(m[u] - base);
        weight += l[u] * f;
#pragma unroll
        for (int c = 0; c < C; ++c)
          sum[c].x += x[u][c].x * f, sum[c].y += x[u][c].y * f, sum[c].z += x[u][c].z * f, sum[c].w += x[u][c].w * f;
      }
    }
    if (lane == 0) s_m[warp] = top, s_l[warp] = weight;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c * 32 + lane < D / 4) s_o[warp][c * 32 + lane] = sum[c];
  }
  __syncthreads();
  if (slot >= mine || slice != 0) return;
  for (int k = 1; k < slices; ++k) top = fmaxf(top, s_m[warp + k]);
  const float base = top == -INFINITY ? 0.0f : top;
  weight = 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) sum[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int k = 0; k < slices; ++k) {
    const float f = fast_exp2(s_m[warp + k] - base);
    weight += s_l[warp + k] * f;
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c * 32 + lane < D / 4) {
        const float4 x = s_o[warp + k][c * 32 + lane];
        sum[c].x += x.x * f, sum[c].y += x.y * f, sum[c].z += x.z * f, sum[c].w += x.w * f;
      }
  }
  const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
  const int64_t out = static_cast<int64_t>(span.x) * p.Hq + (span.y / plan.chunks) * plan.group + chunk * 8 * NT + h;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c * 32 + lane < D / 4)
      reinterpret_cast<uint2*>(static_cast<act_t*>(p.out) + out * D)[c * 32 + lane] =
          make_uint2(pack2<act_t>(sum[c].x * inv, sum[c].y * inv), pack2<act_t>(sum[c].z * inv, sum[c].w * inv));
  if (lane == 0 && p.lse != nullptr) p.lse[out] = weight == 0.0f ? -INFINITY : (top + log2f(weight)) * LN2;
}

int tiles_of(int group) { return group <= 8 ? 1 : 2; }     // n-tiles of eight heads that a warp keeps at once

template <int D>
int full_grid() { return sm_count() * Shape<D>::CTAS; }

int full_grid_of(int D) {
  return D == 64 ? full_grid<64>() : D == 96 ? full_grid<96>() : D == 128 ? full_grid<128>() : D == 192 ? full_grid<192>() : full_grid<256>();
}

// Units that a row of the block table can hold.
int64_t units_of_row(const pla_b200_paged_decode_args& a) { return (static_cast<int64_t>(a.columns) * a.block_size + UNIT - 1) / UNIT; }
// Groups of query heads that share keys and values, over the whole call.
int64_t items_of(const pla_b200_paged_decode_args& a) {
  const int group = a.Hq / a.Hk, at_once = 8 * tiles_of(group);
  return static_cast<int64_t>(a.B) * a.Hk * ((group + at_once - 1) / at_once);
}

// Whether clusters take the call: each item gets one, they fit the SMs at once, and no CTA can get more than 256 KB of rows (the host
// does not know the lengths, but a table row holds no more). Device time with clusters against the other way: one request of 1,024
// tokens of 8 heads of 128 5.7 against 8.7 us, of 4,096 (256 KB) 11.5 against 12.4, of 8,192 18.3 against 13.0; one of 2,048 tokens of 2
// heads of 256 (256 KB) 10.0 against 9.7, 8 ragged ones up to that 11.7 against 14.5.
bool teamed(const pla_b200_paged_decode_args& a) {
  const int64_t unit_bytes = static_cast<int64_t>((a.D + 63) / 64) * UNIT * 128 * 2;
  return items_of(a) * TEAM <= full_grid_of(a.D) && units_of_row(a) <= TEAM * (256 * 1024 / unit_bytes);
}

// CTAs of the other way: no more than there are units, and one per item when no table row holds more than 64 tokens.
int grid_of(const pla_b200_paged_decode_args& a) {
  const int64_t items = items_of(a), per_item = units_of_row(a), full = full_grid_of(a.D);
  const int64_t units = items > 0 && per_item > INT64_MAX / items ? INT64_MAX : items * per_item;
  return static_cast<int>(units < 1 ? 1 : units < full ? units : full);
}

int64_t workspace_bytes(const pla_b200_paged_decode_args& a) {
  if (a.B == 0 || teamed(a)) return 0;
  const int64_t places = 2 * grid_of(a);
  return places * static_cast<int64_t>(sizeof(int4)) + places * 8 * tiles_of(a.Hq / a.Hk) * (a.D + 2) * 4;
}

// Tensor map of one cache: [page][token][head][channel], boxes of TILE tokens and 64 channels of one head. Axes of one entry get
// any valid stride: their index is always 0.
int cache_map(CUtensorMap* map, const pla_b200_paged_decode_args& a, void* base, const pla_b200_page_strides& st) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void*> found{nullptr};
  void* fn = found.load(std::memory_order_acquire);
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult how;
    PLA_CUDA_OK(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how));
    PLA_REQUIRE(fn != nullptr && how == cudaDriverEntryPointSuccess, PLA_B200_E_CUDA, "the driver has no cuTensorMapEncodeTiled");
    found.store(fn, std::memory_order_release);
  }
  auto bytes = [&](int64_t n, int64_t stride) { return static_cast<cuuint64_t>(n <= 1 ? a.D : stride) * 2; };
  const cuuint64_t size[4] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.Hk), static_cast<cuuint64_t>(a.block_size),
                              static_cast<cuuint64_t>(a.num_blocks)};
  const cuuint64_t stride[3] = {bytes(a.Hk, st.head), bytes(a.block_size, st.token), bytes(a.num_blocks, st.block)};
  const cuuint32_t box[4] = {64, 1, TILE, 1}, step[4] = {1, 1, 1, 1};
  // Rows of whole 256-byte pieces are fetched in these (one request of 128K tokens of 128 channels 93.5 -> 91.4 us); others would
  // bring a neighbour's bytes along (D = 192: 81.3 -> 82.8 us).
  const CUtensorMapL2promotion fetch = a.D % 128 == 0 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
  const CUresult rc = reinterpret_cast<Encode>(fn)(
      map, a.act_dtype == PLA_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, size, stride, box, step,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, fetch, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PLA_REQUIRE(rc == CUDA_SUCCESS, PLA_B200_E_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(rc));
  return PLA_B200_OK;
}

// Strides that a tensor map can hold; pages of whole tiles.
bool boxed(const pla_b200_paged_decode_args& a) {
  auto fits = [&](const pla_b200_page_strides& s) {
    auto ok = [](int64_t n, int64_t stride) { return n <= 1 || (stride > 0 && stride < int64_t{1} << 38); };
    return ok(a.num_blocks, s.block) && ok(a.block_size, s.token) && ok(a.Hk, s.head);
  };
  return a.block_size % TILE == 0 && a.num_blocks > 0 && a.num_blocks <= INT32_MAX && fits(a.k_strides) && fits(a.v_strides);
}

template <typename act_t, int D, int NT, bool BOXED, bool TEAMED>
int launch(const pla_b200_paged_decode_args& a, cudaStream_t stream) {
  using S = Shape<D>;
  static DeviceOnce once;
  int dev = 0;
  PLA_CUDA_OK(cudaGetDevice(&dev));
  if (once.needed(dev)) {
    PLA_CUDA_OK(cudaFuncSetAttribute(paged_decode_kernel<act_t, D, NT, BOXED, TEAMED>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    once.mark(dev);
  }
  Plan plan = {};
  plan.page = Divisor(static_cast<uint32_t>(a.block_size));
  plan.group = a.Hq / a.Hk;
  plan.chunks = (plan.group + 8 * NT - 1) / (8 * NT);
  if constexpr (TEAMED) {
    plan.grid = static_cast<int>(items_of(a) * TEAM);
  } else {
    plan.grid = grid_of(a);
    const int64_t places = 2 * plan.grid;
    plan.spans = static_cast<int4*>(a.workspace);
    plan.part_o = reinterpret_cast<float*>(plan.spans + places);
    plan.part_m = plan.part_o + places * 8 * NT * D;
    plan.part_l = plan.part_m + places * 8 * NT;
  }
  CUtensorMap k_map = {}, v_map = {};
  if constexpr (BOXED) {
    int rc = cache_map(&k_map, a, const_cast<void*>(a.k_cache), a.k_strides);
    if (rc == PLA_B200_OK) rc = cache_map(&v_map, a, const_cast<void*>(a.v_cache), a.v_strides);
    if (rc != PLA_B200_OK) return rc;
  }
  if constexpr (TEAMED) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.grid);
    cfg.blockDim = dim3(THREADS + 32 * LOADERS<D, NT, BOXED>);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = TEAM;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PLA_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_decode_kernel<act_t, D, NT, BOXED, TEAMED>, a, plan, k_map, v_map));
    return PLA_B200_OK;
  }
  paged_decode_kernel<act_t, D, NT, BOXED, TEAMED><<<plan.grid, THREADS + 32 * LOADERS<D, NT, BOXED>, S::SMEM, stream>>>(a, plan, k_map, v_map);
  PLA_CUDA_OK(cudaGetLastError());
  if (units_of_row(a) > 1) {                        // else every item is one unit and was stored whole
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * plan.grid);
    cfg.blockDim = dim3(JOIN_WARPS * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    PLA_CUDA_OK(cudaLaunchKernelEx(&cfg, paged_join_kernel<act_t, D, NT>, a, plan));
  }
  return PLA_B200_OK;
}

template <typename act_t, int D, int NT>
int launch_tiles(const pla_b200_paged_decode_args& a, cudaStream_t s) {
  if (teamed(a)) return boxed(a) ? launch<act_t, D, NT, true, true>(a, s) : launch<act_t, D, NT, false, true>(a, s);
  return boxed(a) ? launch<act_t, D, NT, true, false>(a, s) : launch<act_t, D, NT, false, false>(a, s);
}

template <typename act_t, int D>
int launch_size(const pla_b200_paged_decode_args& a, cudaStream_t s) {
  return tiles_of(a.Hq / a.Hk) == 1 ? launch_tiles<act_t, D, 1>(a, s) : launch_tiles<act_t, D, 2>(a, s);
}

template <typename act_t>
int launch_for(const pla_b200_paged_decode_args& a, cudaStream_t s) {
  switch (a.D) {
    case 64: return launch_size<act_t, 64>(a, s);
    case 96: return launch_size<act_t, 96>(a, s);
    case 128: return launch_size<act_t, 128>(a, s);
    case 192: return launch_size<act_t, 192>(a, s);
    default: return launch_size<act_t, 256>(a, s);
  }
}

bool head_size_ok(int D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }
bool strides16(const pla_b200_page_strides& s) { return s.block % 8 == 0 && s.token % 8 == 0 && s.head % 8 == 0; }

}  // namespace
}  // namespace pla

namespace pla {
namespace {

int check_sizes(const pla_b200_paged_decode_args& a) {
  PLA_REQUIRE(a.B >= 0 && a.Hq > 0 && a.Hk > 0 && a.Hq % a.Hk == 0, PLA_B200_E_INVALID,
              "paged decode needs B >= 0 and a positive number of query heads that the key/value heads divide");
  PLA_REQUIRE(head_size_ok(a.D), PLA_B200_E_UNSUPPORTED, "the head size must be 64, 96, 128, 192 or 256");
  PLA_REQUIRE(static_cast<int64_t>(a.B) * a.Hq <= INT32_MAX, PLA_B200_E_TOO_LARGE, "too many rows");
  PLA_REQUIRE(a.columns >= 0 && a.block_size > 0 && a.num_blocks >= 0, PLA_B200_E_INVALID, "bad block table sizes");
  return PLA_B200_OK;
}

}  // namespace
}  // namespace pla

extern "C" int64_t pla_b200_paged_decode_workspace_bytes(const pla_b200_paged_decode_args* args) {
  using namespace pla;
  PLA_REQUIRE(args != nullptr, PLA_B200_E_INVALID, "args is NULL");
  const int rc = check_sizes(*args);
  return rc != PLA_B200_OK ? rc : workspace_bytes(*args);
}

extern "C" int pla_b200_paged_decode(const pla_b200_paged_decode_args* args, void* stream) {
  using namespace pla;
  PLA_REQUIRE(args != nullptr, PLA_B200_E_INVALID, "args is NULL");
  pla_b200_paged_decode_args a = *args;
  default_status(a);
  const int rc = check_sizes(a);
  if (rc != PLA_B200_OK) return rc;
  PLA_REQUIRE(a.act_dtype == PLA_B200_BF16 || a.act_dtype == PLA_B200_F16, PLA_B200_E_INVALID, "paged decode takes bf16 or fp16");
  if (a.B == 0) return PLA_B200_OK;
  PLA_REQUIRE(a.q && a.out && a.seq_lens && (a.columns == 0 || a.block_table) && (a.num_blocks == 0 || (a.k_cache && a.v_cache)),
              PLA_B200_E_INVALID, "q, the caches, block_table, seq_lens and out are required");
  const int64_t bytes = workspace_bytes(a);
  PLA_REQUIRE(bytes == 0 || (a.workspace && a.workspace_bytes >= bytes), PLA_B200_E_INVALID, "the workspace is missing or too small");
  PLA_REQUIRE(aligned16(a.q) && aligned16(a.k_cache) && aligned16(a.v_cache) && aligned16(a.out) && aligned16(a.workspace) && a.q_row_stride % 8 == 0 &&
                  a.q_head_stride % 8 == 0 && strides16(a.k_strides) && strides16(a.v_strides),
              PLA_B200_E_ALIGN, "q, out, workspace and cache rows must be 16-byte aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a.act_dtype == PLA_B200_BF16 ? launch_for<__nv_bfloat16>(a, s) : launch_for<__half>(a, s);
}
