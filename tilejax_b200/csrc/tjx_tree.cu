// Attention of a tree of drafted tokens over the ragged paged cache: the decode case of ragged paged attention
// (examples/ragged_paged_attention.py:121-149) for sequences that bring several tokens of which each sees the cached
// prefix and those of its own sequence that its mask names (its ancestors in the tree, and itself).
//   o[t, h] = sum_p softmax_p(sm_scale q[t, h] . k[p, h / group]) v[p, h / group]
// over the positions p < kv_len - q_len and the nodes j (position kv_len - q_len + j) with bit j of tree_mask[t] set.
//
// The rows (node, query head) that share a KV head share its cache, so a position costs 512 bytes of HBM and, at 128
// rows of tensor work however few are used, 33 k multiply-adds: 11.6 ns of one SM's share of the memory rate against
// 5.8 of its tensor rate. So one kernel serves one node and many: whole 128-row tcgen05 tiles, padded.
//
// A unit is (sequence, KV head, up to 256 rows): its rows make one tile of 128, or two that share every K / V block of
// 64 positions. The units' blocks, in order and weighed by what they cost, are cut into equal runs, one for each CTA: a
// CTA walks the end of one unit, whole units, and the beginning of another, and what it has of a unit that others share
// is a partial result (running maximum, sum, unnormalised rows) that tree_join_kernel joins in order. One persistent CTA
// per SM:
//
//   warps 0, 11 producers: TMA loads of Q (a buffer per row tile) and K blocks, and of V blocks, into rings (boxes of at
//               most a page)
//   warps 1, 2  MMA issuers, one for each group: S = Q K^T one job ahead of O += P V, P read from TMEM
//   warps 3-6   softmax of the one group, warps 7-10 of the other (a thread owns a row)
//
// A job is (row tile, block). With two row tiles each group (an issuer and its four softmax warps) has one of them; with
// one tile the groups take the even and the odd blocks and each keep a running maximum, sum and output over theirs,
// which they join in TMEM at the end of the unit. TMEM: each group has two score buffers of 64 columns (P, bf16, overlays
// the scores), so that the next scores are made while it works, and 128 columns of output.
//
// What it reaches: one token a sequence over 64 caches of 1000 to 8100 positions 191 us on pages of 128 and 193 on pages of 16,
// 6.2 TB/s of the cache; trees of 16 over 32 caches of up to 4096 61 us; trees of 64 (both row tiles full) over two caches of
// 125 k 266 us, 0.97 PFLOP/s, and 317 us repeated: then the GPU is at its power limit (1000 W, 1.5 GHz).
// There blocks of 128 positions (whose scores' products read Q from shared memory half as often: 512 cycles for 832, but
// one score buffer a group) took the same time, repeated and alone, and so did all exponentials on one pipe. What a unit
// takes beside its blocks is to a large part code that is not in the instruction cache when its turn comes: a seventh less of
// it made every call shorter, by 3 to 5 %.
//
// A wait tells a barrier's phase from the one before it only. So whoever waits on a ring slot must have seen its use
// before: rings have an even number of slots and blocks keep their parity over the whole run, so that a group finds
// its blocks in the same slots always.
#include <algorithm>
#include <type_traits>

#include "tjx_host.cuh"
#include "tjx_ptx.cuh"

#include "../../include/tilejax_b200.h"

namespace tjx {

constexpr int TR_D = 128;
constexpr int TR_ROWS = 128;   // rows of a tile
constexpr int TR_BLOCK = 64;   // positions of a block
constexpr int TR_K_STAGES = 4;
constexpr int TR_V_STAGES = 6;  // a V block is held longer: until its probabilities are made
constexpr int TR_THREADS = 384;
constexpr float TR_LOG2E = 1.4426950408889634f;
// The running maximum (log2 units) of a row that has seen no score above minus infinity: the lowest number, so that no score
// is below it. Its sum tells whether it has seen one at all: 0 if not, else something.
constexpr float TR_NOTHING = -3.402823466e38f;
// From this maximum on (log2 units) a row's scores are rounded before the maximum is taken off. Below it that is one fused
// step, which is more exact but leaves the maximum's own rounding in every exponent (at most 8 here): the same for all of the
// row, so gone after the division by the sum, unless it leaves f32's range, as it would from some 2^31 on.
constexpr float TR_FAR = 268435456.f;
constexpr float TR_RESCALE = 8.0f;    // raise the running maximum only for a gain of 2^8: the same result, rarely a rescale
// What a run is cut by, in units of about 300 cycles: a block of one row tile (bound by its loads, 1230 cycles), of two
// (by their softmax, 1950), and what a unit takes beside its blocks: the last scores masked and their V rows looked at, the
// pipeline drained, the rows out. Without the weights the CTA with the most units, or with the widest, runs longer
// than the others (trees of 16 over 32 caches of up to 4096: 69.5 -> 61.5 us; of up to 64 over 64 of up to 8100: 325 -> 289).
constexpr int TR_COST_ONE = 4, TR_COST_TWO = 6, TR_COST_UNIT = 32;
constexpr int TR_MIN_SHARE = 8;  // a run's cost, at least: two blocks of one row tile, one a group (one sequence 11.8 us with 12, 11.0; 11.5 with 6)
static_assert(TR_MIN_SHARE >= TR_COST_TWO && TR_MIN_SHARE >= TR_COST_ONE, "every run inside a unit has a block");

struct TreeParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const __nv_bfloat16* kv_cache;
  const int32_t *kv_lens, *page_indices, *cu_q_lens, *tree_mask, *distribution;
  int T, S, H, Hkv, group, page_size, pages_per_seq, num_pages, words;
  int tile_nodes;  // nodes of a row tile: 128 / group
  int box_rows;    // positions of one TMA box: the largest power of two that divides the page size, at most 64
  float scale_log2e;
  double per_cta;    // 1 / CTAs
  int part_rows;     // rows of a partial result
  float4* part_o;    // [2 CTAs][32][part_rows]: four columns of a row (a warp's rows lie side by side)
  float2* part_ml;   // [2 CTAs][part_rows]: running maximum (log2 units) and sum
  int4* joins;       // [CTAs]: the unit that starts in CTA c and ends in a later one: first token, nodes, KV head, last CTA
  int* status;
};

struct TreeSmem {
  static constexpr int Q_BYTES = TR_ROWS * TR_D * 2;   // two halves of 64 columns
  static constexpr int KV_BYTES = TR_BLOCK * TR_D * 2;
  static constexpr int Q_OFF = 0;  // two buffers
  static constexpr int K_OFF = 2 * Q_BYTES;
  static constexpr int V_OFF = K_OFF + TR_K_STAGES * KV_BYTES;
  static constexpr int STAT_OFF = V_OFF + TR_V_STAGES * KV_BYTES;  // float2[2][128]: maximum and sum of each group's rows
  static constexpr int BAD_OFF = STAT_OFF + 2 * TR_ROWS * 8;       // uint32[2 groups][2][4]: rows of V that are not finite
  static constexpr int SCAN_OFF = BAD_OFF + 64;                    // long long[12], and int[10]: where this CTA starts
  static constexpr int BAR_OFF = SCAN_OFF + 96 + 40;
  static constexpr int N_BARS = 21 + 2 * TR_K_STAGES + 2 * TR_V_STAGES;
  static constexpr int TOTAL = BAR_OFF + 8 * N_BARS + 16;
};
static_assert(TR_K_STAGES % 2 == 0 && TR_V_STAGES % 2 == 0, "a slot's blocks are of one parity");
static_assert(TreeSmem::TOTAL <= 232448, "shared memory of one CTA");

// One sequence's sizes, clamped to what the arrays hold.
struct TreeSeq {
  int tok0, q_len, ctx, end, blocks, pairs;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int c0, int c1, int len) {
  TreeSeq r;
  r.tok0 = min(max(c0, 0), p.T);
  r.q_len = max(min(c1, p.T) - r.tok0, 0);
  r.end = min(max(len, 0), p.pages_per_seq * p.page_size);  // positions to walk
  r.ctx = len < 0 ? -r.q_len : len - r.q_len;               // position of node 0
  r.blocks = max((r.end + TR_BLOCK - 1) / TR_BLOCK, 1);     // (one where there is nothing: its rows become zero)
  r.pairs = (r.q_len + 2 * p.tile_nodes - 1) / (2 * p.tile_nodes);
  return r;
}

__device__ __forceinline__ TreeSeq tree_seq(const TreeParams& p, int s) {
  return tree_seq(p, p.cu_q_lens[s], p.cu_q_lens[s + 1], p.kv_lens[s]);
}

// a / b for a >= 0, b > 0: a 64-bit division only where it takes one.
__device__ __forceinline__ long long tree_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// What the units of one KV head of a sequence cost, and one unit of two row tiles.
__device__ __forceinline__ long long tree_pair_cost(const TreeSeq& q) {
  return TR_COST_UNIT + static_cast<long long>(q.blocks) * TR_COST_TWO;
}
__device__ __forceinline__ int tree_block_cost(const TreeParams& p, const TreeSeq& q, int pr) {
  return q.q_len - pr * 2 * p.tile_nodes > p.tile_nodes ? TR_COST_TWO : TR_COST_ONE;
}
__device__ __forceinline__ long long tree_head_cost(const TreeParams& p, const TreeSeq& q) {
  return q.pairs == 0 ? 0
                      : (q.pairs - 1) * tree_pair_cost(q) + TR_COST_UNIT +
                            static_cast<long long>(q.blocks) * tree_block_cost(p, q, q.pairs - 1);
}

// A CTA's walk over its run: the same in every role. Block j of a unit costs its weight from TR_COST_UNIT + j * weight
// on and is of the run that this falls into.
struct TreePortion {
  int s, tok, nodes;     // first token and nodes of the unit
  int hk, ctx, end;
  int j0, j1;            // blocks of the unit
  bool whole, starts;    // all of the unit's blocks; its first block among them
  bool two;              // two row tiles
  int past;              // of a unit that ends in a later run: where its last block starts, seen from the end of this one
};
// x / weight for x >= 0.
__device__ __forceinline__ int tree_per_weight(int x, bool two) {
  return static_cast<int>(two ? static_cast<uint32_t>(x) / TR_COST_TWO : static_cast<uint32_t>(x) / TR_COST_ONE);
}
struct TreeWalk {
  int s, hk, pr;
  int at;          // of the unit's cost (at most 2^31 / 64 blocks), where the walk stands
  long long left;  // of the run's, what is left
  TreeSeq q;
  __device__ __forceinline__ void load(const TreeParams& p) {  // by whole warps: the same values, and said to be so
    q = tree_seq(p, s);
    q.tok0 = __shfl_sync(0xFFFFFFFFu, q.tok0, 0), q.q_len = __shfl_sync(0xFFFFFFFFu, q.q_len, 0);
    q.ctx = __shfl_sync(0xFFFFFFFFu, q.ctx, 0), q.end = __shfl_sync(0xFFFFFFFFu, q.end, 0);
    q.blocks = __shfl_sync(0xFFFFFFFFu, q.blocks, 0), q.pairs = __shfl_sync(0xFFFFFFFFu, q.pairs, 0);
  }
  __device__ __forceinline__ bool next(const TreeParams& p, TreePortion& o) {
    while (left > 0) {
      const int weight = tree_block_cost(p, q, pr), node0 = pr * 2 * p.tile_nodes;
      const int cost = TR_COST_UNIT + q.blocks * weight;
      const bool ends = left >= cost - at;
      const int to = ends ? cost : at + static_cast<int>(left);
      o.s = s, o.hk = hk, o.ctx = q.ctx, o.end = q.end;
      o.tok = q.tok0 + node0;
      o.nodes = min(q.q_len - node0, 2 * p.tile_nodes);
      o.two = o.nodes > p.tile_nodes;
      o.j0 = tree_per_weight(max(at - TR_COST_UNIT, 0) + weight - 1, o.two);
      o.j1 = ends ? q.blocks : tree_per_weight(max(to - TR_COST_UNIT, 0) + weight - 1, o.two);
      o.starts = o.j0 == 0, o.whole = o.starts && o.j1 == q.blocks;
      o.past = cost - weight - to;
      left -= cost - at, at = 0;
      if (++pr == q.pairs) {
        pr = 0;
        if (++hk == p.Hkv) {
          hk = 0;
          if (left > 0) {
            do ++s, load(p); while (q.pairs == 0);  // (something is left, so a sequence with a unit follows)
          }
        }
      }
      if (o.j1 > o.j0) return true;
    }
    return false;
  }
};

// 32 positions from `pos` on as a row sees them: its mask's bits from node pos - ctx on, ones before the first node,
// zeros past the mask's words and from `end` on.
struct TreeMask {  // a row's mask, its first two words fetched ahead
  const int32_t* row;
  int words;
  uint32_t first, second;
  __device__ __forceinline__ uint32_t word(int w) const {
    return w < 0 ? 0xFFFFFFFFu : w == 0 ? first : w == 1 ? second : w < words ? static_cast<uint32_t>(row[w]) : 0u;
  }
};
__device__ __forceinline__ uint32_t tree_bits(const TreeMask& mask, int pos, int ctx, int end) {
  uint32_t bits = 0xFFFFFFFFu;
  if (pos + 32 > ctx) {
    const int o = pos - ctx, w = o >> 5, shift = o & 31;  // (arithmetic shift: w = -1 or less before the nodes)
    bits = __funnelshift_r(mask.word(w), mask.word(w + 1), shift);
  }
  const int valid = end - pos;
  return valid >= 32 ? bits : valid <= 0 ? 0u : bits & ((1u << valid) - 1u);
}

// Whether a table entry is a page. A position whose entry is not (the planner's -1 where it had none left) is seen by no row. Its
// copies start behind the cache, which makes its keys NaN and its values zero: its score says so by itself, and nobody has
// to look the table over beforehand (done by the producers, a vote a block, single tokens took a tenth longer). Whoever
// meets a score that is NaN looks the block's entries up.
__device__ __forceinline__ bool tree_is_page(const TreeParams& p, int entry) {
  return static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.num_pages);
}

// Bits of the positions of the block at kv0 that have a page (by a whole warp; pages end at multiples of 16).
__device__ __forceinline__ uint2 tree_paged(const TreeParams& p, int s, int kv0) {
  const int lane = threadIdx.x & 31;
  bool paged = false;
  if (lane < TR_BLOCK / 16) {
    const int entry = min((kv0 + 16 * lane) / p.page_size, p.pages_per_seq - 1);
    paged = tree_is_page(p, p.page_indices[static_cast<size_t>(s) * p.pages_per_seq + entry]);
  }
  const uint32_t v = __ballot_sync(0xFFFFFFFFu, paged);
  return make_uint2((v & 1 ? 0xFFFFu : 0u) | (v & 2 ? 0xFFFF0000u : 0u), (v & 4 ? 0xFFFFu : 0u) | (v & 8 ? 0xFFFF0000u : 0u));
}

// A whole warp's bounded wait, with one outcome for all lanes; a phase that is there already costs one test and one vote.
__device__ __forceinline__ bool tree_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (__builtin_expect(__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity) != 0), 1)) return true;
  return __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity, abort_flag, status, code)) != 0;
}

__device__ __forceinline__ bool tree_far(float m) { return fabsf(m) >= TR_FAR && m != TR_NOTHING; }

// What a row's products are weighed by: zero where it sees nothing, NaN where it sees minus infinity only (0 / 0 by the formula).
__device__ __forceinline__ float tree_inverse(float m, float sum) {
  return sum == 0.f ? 0.f : m == TR_NOTHING ? NAN : 1.0f / sum;
}

// Zero times every element, added up: NaN where one is not finite.
__device__ __forceinline__ void tree_zeros(__nv_bfloat162& sum, uint32_t x) {
  sum = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f), sum);
}

__global__ void __launch_bounds__(TR_THREADS, 1)
    tree_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const TreeParams p) {
  using L = TreeSmem;
  extern __shared__ __align__(1024) uint8_t base_ptr[];
  const uint32_t base = smem_u32(base_ptr);
  if ((base & 1023u) != 0) {  // (the tiles' swizzle goes by address bits; the runtime puts the array at 1024)
    if (threadIdx.x == 0) {
      atomicCAS(p.status, 0, TJX_ERR_WAIT_OTHER);
      p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    return;
  }
  // (Under way while the barriers are set up; without waiting for the number of sequences.)
  const int per_thread = (p.S + TR_THREADS - 1) / TR_THREADS;
  const int s_lo = min(static_cast<int>(threadIdx.x) * per_thread, p.S), s_hi = min(s_lo + per_thread, p.S);
  int c0_lo = 0, c1_lo = 0, len_lo = 0;
  if (s_lo < s_hi) c0_lo = p.cu_q_lens[s_lo], c1_lo = p.cu_q_lens[s_lo + 1], len_lo = p.kv_lens[s_lo];
  const int distribution = p.distribution[0];
  const uint32_t bar = base + L::BAR_OFF;
  auto q_full = [&](int b) { return bar + 8u * b; };
  auto q_empty = [&](int b) { return bar + 8u * (2 + b); };
  auto s_full = [&](int t, int b) { return bar + 8u * (4 + 2 * t + b); };
  auto p_ready = [&](int t, int b) { return bar + 8u * (8 + 2 * t + b); };
  auto o_done = [&](int t, int b) { return bar + 8u * (12 + 2 * t + b); };
  auto v_seen = [&](int t) { return bar + 8u * (16 + t); };  // a group's warps have looked at a V block
  const uint32_t v_seen_both = bar + 8u * 18;
  const uint32_t stats_ready = bar + 8u * 19, outputs_read = bar + 8u * 20;
  constexpr int RING = 21;
  auto k_full = [&](int i) { return bar + 8u * (RING + i); };
  auto k_empty = [&](int i) { return bar + 8u * (RING + TR_K_STAGES + i); };
  auto v_full = [&](int i) { return bar + 8u * (RING + 2 * TR_K_STAGES + i); };
  auto v_empty = [&](int i) { return bar + 8u * (RING + 2 * TR_K_STAGES + TR_V_STAGES + i); };
  constexpr int N_BARS = L::N_BARS;
  static_assert(N_BARS == RING + 2 * TR_K_STAGES + 2 * TR_V_STAGES, "");
  volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(base_ptr + L::BAR_OFF + 8 * N_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + L::BAR_OFF + 8 * N_BARS + 8);
  volatile long long* scan = reinterpret_cast<volatile long long*>(base_ptr + L::SCAN_OFF);
  float2* stats = reinterpret_cast<float2*>(base_ptr + L::STAT_OFF);
  volatile uint32_t* bad_rows = reinterpret_cast<volatile uint32_t*>(base_ptr + L::BAD_OFF);

  const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x < N_BARS) {
    // p_ready, v_seen: the warps of a group; the next three: of both. A Q, K or V buffer is free when both groups say
    // so (where only one uses it, the producer speaks for the other).
    const int i = threadIdx.x;
    const bool by_both = i == 2 || i == 3 || (i >= RING + TR_K_STAGES && i < RING + 2 * TR_K_STAGES) ||
                         i >= RING + 2 * TR_K_STAGES + TR_V_STAGES;
    mbar_init(bar + 8u * i, (i >= 8 && i < 12) || i == 16 || i == 17 ? 4 : i >= 18 && i < RING ? 8 : by_both ? 2 : 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_holder)), 512);
    tmem_relinquish();
  }
  // All costs added up, and where this CTA's run starts: a thread takes consecutive sequences, the thread that has the
  // run's first block finds its sequence.
  volatile int* start = reinterpret_cast<volatile int*>(base_ptr + L::SCAN_OFF + 96);
  auto cost_of = [&](const TreeSeq& q) { return tree_head_cost(p, q) * p.Hkv; };
  long long mine = 0;
  TreeSeq q_lo{};
  for (int s = s_lo; s < s_hi; ++s) {
    const TreeSeq q = s == s_lo ? tree_seq(p, c0_lo, c1_lo, len_lo) : tree_seq(p, s);
    if (s == s_lo) q_lo = q;
    mine += s < distribution ? cost_of(q) : 0;
  }
  long long upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += y;
  }
  if (lane == 31) scan[warp] = upto;
  __syncthreads();
  long long total = 0;
  const int scans = min((p.S + 31) / 32, TR_THREADS / 32);  // at least the warps with a sequence
#pragma unroll 1
  for (int w = 0; w < scans; ++w) {
    if (w == warp) upto += total;
    total += scan[w];
  }
  // (At least total / CTAs, whichever way the product was rounded.)
  const long long share = max(static_cast<long long>(static_cast<double>(total) * p.per_cta) + 1, static_cast<long long>(TR_MIN_SHARE));
  const long long first = share * blockIdx.x, count = min(share, total - first);  // (count <= 0: nothing)
  if (count > 0 && first >= upto - mine && first < upto) {
    long long off = first - (upto - mine);
    int s = s_lo;
    TreeSeq q = q_lo;
    for (long long n; off >= (n = cost_of(q)); q = tree_seq(p, ++s)) off -= n;
    start[0] = s, start[1] = q.tok0, start[2] = q.q_len, start[3] = q.ctx, start[4] = q.end, start[5] = q.blocks;
    start[6] = q.pairs, start[7] = static_cast<int>(off), start[8] = static_cast<int>(off >> 32);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, *tmem_holder, 0);
  // (Through shuffles: the compiler must know that a warp's lanes walk together, or it keeps the issuers' addresses and
  // loop counters per lane.)
  TreeWalk walk;
  {
    const int word = lane < 9 ? start[lane] : 0;
    auto get = [&](int i) { return __shfl_sync(0xFFFFFFFFu, word, i); };
    walk.s = get(0), walk.hk = 0, walk.pr = 0, walk.at = 0, walk.left = __shfl_sync(0xFFFFFFFFu, count, 0);
    walk.q.tok0 = get(1), walk.q.q_len = get(2), walk.q.ctx = get(3), walk.q.end = get(4), walk.q.blocks = get(5);
    walk.q.pairs = get(6);
    long long off = static_cast<long long>(static_cast<uint32_t>(get(7))) | (static_cast<long long>(get(8)) << 32);
    if (walk.left > 0) {  // (else nothing was found)
      // The KV head, and the unit of it: counted by the lanes, 32 at a time, each of which costs the same.
      const long long head = tree_head_cost(p, walk.q), pair = tree_pair_cost(walk.q);
      for (int n = 32; n == 32; walk.hk += n) n = __popc(__ballot_sync(0xFFFFFFFFu, (walk.hk + lane + 1) * head <= off));
      off -= walk.hk * head;
      for (int n = 32; n == 32; walk.pr += n)
        n = __popc(__ballot_sync(0xFFFFFFFFu, walk.pr + lane + 1 < walk.q.pairs && (walk.pr + lane + 1) * pair <= off));
      walk.at = static_cast<int>(off - walk.pr * pair);
    }
  }

  if (warp == 0 || warp == 11) {
    // ------------------------------------------------------------------ producers: of Q and K, of V
    const bool keys = warp == 0;
    const CUtensorMap* map = keys ? &map_k : &map_v;
    bool ok = true;
    int qc = 0;      // Q tiles loaded so far
    int block = 0;   // blocks loaded so far
    const int boxes = TR_BLOCK / p.box_rows;
    const uint32_t box_bytes = p.box_rows * 128;
    const bool looks = lane < boxes;  // lane l looks up the page of box l
    auto wait = [&](uint32_t b, uint32_t parity) {
      return tree_wait(b, parity, abort_flag, p.status, TJX_ERR_WAIT_EMPTY);
    };
    TreePortion u;
    while (ok && walk.next(p, u)) {
      const int32_t* table = p.page_indices + static_cast<size_t>(u.s) * p.pages_per_seq;
      // The page of this lane's box of block j, and the box's first row there: fetched a block ahead. (An entry past the
      // table is clamped: its positions are past the sequence's end.)
      int page = 0, page_row = 0;
      auto fetch = [&](int j) {
        const int pos = j * TR_BLOCK + lane * p.box_rows;
        const int entry = pos / p.page_size;
        page = table[min(entry, p.pages_per_seq - 1)], page_row = pos - entry * p.page_size;
      };
      if (looks) fetch(u.j0);
      if (keys) {
        for (int r = 0; r < (u.two ? 2 : 1) && ok; ++r, ++qc) {
          const int b = qc & 1;
          ok = wait(q_empty(b), ((qc >> 1) & 1) ^ 1u);
          if (!ok) break;
          if (lane == 0) {
            const uint32_t dst = base + L::Q_OFF + b * L::Q_BYTES;
            mbar_expect_tx(q_full(b), static_cast<uint32_t>(p.tile_nodes * p.group) * 256u);
            const int tok = u.tok + r * p.tile_nodes;
            tma_load_3d(dst, &map_q, 0, u.hk * p.group, tok, q_full(b));
            tma_load_3d(dst + L::Q_BYTES / 2, &map_q, 64, u.hk * p.group, tok, q_full(b));
            if (u.two) mbar_arrive(q_empty(b));  // one group uses it
          }
          __syncwarp();
        }
      }
      for (int j = u.j0; j < u.j1 && ok; ++j, ++block) {
        const int row = tree_is_page(p, page) ? page * p.page_size + page_row : p.num_pages * p.page_size;  // (the latter: behind the cache)
        if (looks && j + 1 < u.j1) fetch(j + 1);
        const int slot = block % (keys ? TR_K_STAGES : TR_V_STAGES), use = block / (keys ? TR_K_STAGES : TR_V_STAGES);
        const uint32_t full = keys ? k_full(slot) : v_full(slot), empty = keys ? k_empty(slot) : v_empty(slot);
        // One lane issues the block's copies, with coordinates that the compiler knows to be the same in every lane. A copy
        // per lane took the warp a turn for each, some 100 cycles, and on pages of 16, with eight a block, the producers were
        // what the kernel waited for (trees of 16 over 64 caches of up to 8100 positions: 223 -> 210 us).
        int rows[TR_BLOCK / 16];
#pragma unroll
        for (int i = 0; i < TR_BLOCK / 16; ++i) rows[i] = __shfl_sync(0xFFFFFFFFu, row, i);
        const uint32_t dst = base + (keys ? L::K_OFF : L::V_OFF) + slot * L::KV_BYTES;
        const int head = 2 * u.hk + (keys ? 0 : 1);
        ok = wait(empty, (use & 1) ^ 1u);
        if (!ok) break;
        if (elect_one()) {
          mbar_expect_tx(full, L::KV_BYTES);
          if (!u.two) mbar_arrive(empty);
#pragma unroll
          for (int i = 0; i < TR_BLOCK / 16; ++i) {
            if (i >= boxes) break;
            tma_load_3d(dst + i * box_bytes, map, 0, head, rows[i], full);
            tma_load_3d(dst + i * box_bytes + L::KV_BYTES / 2, map, 64, head, rows[i], full);
          }
        }
        __syncwarp();
      }
    }
    __syncwarp();
  } else if (warp <= 2) {
    // ------------------------------------------------------------------ MMA issuers (whole warps; one lane issues)
    // One issuer for both groups was the kernel's limit: some 1700 cycles a job, of which a tile's MMAs are 600 and the
    // rest waits that find their barrier ready, descriptors and commits, one after the other.
    const int t = warp - 1;
    const uint32_t idesc_qk = idesc_bf16_f32(128, TR_BLOCK, 0, 0);  // Q and K both K-major
    const uint32_t idesc_pv = idesc_bf16_f32(128, TR_D, 0, 1);      // P from TMEM, V MN-major
    auto wait = [&](uint32_t b, uint32_t parity, int code) {
      return tree_wait(b, parity, abort_flag, p.status, code);
    };
    // A group's blocks of a portion: all of them, or with one row tile those of its parity, counted over the run.
    auto first_of = [&](const TreePortion& u, int before) { return u.two ? 0 : (t - before) & 1; };
    TreeWalk ahead = walk;  // the scores' walk runs ahead of the outputs'
    TreePortion a{}, b{};
    int ia = 0, ib = 0;              // block of the portion
    int a_blocks = 0, b_blocks = 0;  // blocks of the portions before
    int ca = 0, cb = 0;              // jobs issued so far
    int qc = 0;                      // Q tiles of the portions before
    bool ok = true, more = true;
    while (ok) {
      while (ok && more && ia >= a.j1 - a.j0) {  // (a portion of one block has none for one of the groups)
        a_blocks += a.j1 - a.j0, qc += a.nodes == 0 ? 0 : a.two ? 2 : 1;
        more = ahead.next(p, a);
        if (!more) break;
        ia = first_of(a, a_blocks);
        for (int q = qc; q < qc + (a.two ? 2 : 1) && ok; ++q) ok = wait(q_full(q & 1), (q >> 1) & 1, TJX_ERR_WAIT_FULL);
        if (ok && ia >= a.j1 - a.j0 && elect_one()) mbar_arrive(q_empty(qc & 1));
      }
      if (!ok) break;
      if (more) {
        // Q K^T
        const int block = a_blocks + ia, q_buffer = (qc + (a.two ? t : 0)) & 1;
        const int ks = block % TR_K_STAGES;
        ok = wait(k_full(ks), (block / TR_K_STAGES) & 1, TJX_ERR_WAIT_FULL);
        if (!ok) break;
        tc_fence_after_sync();
        const uint32_t qa = base + L::Q_OFF + q_buffer * L::Q_BYTES, ka = base + L::K_OFF + ks * L::KV_BYTES;
        const uint64_t q0 = smem_desc_sw128(qa, 16, 1024), k0 = smem_desc_sw128(ka, 16, 1024);
        uint64_t qd[8], kd[8];
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qd[kk] = q0 + (((kk >> 2) * (L::Q_BYTES / 2) + (kk & 3) * 32) >> 4);
          kd[kk] = k0 + (((kk >> 2) * (L::KV_BYTES / 2) + (kk & 3) * 32) >> 4);
        }
        mma_ss_x8_commit(tmem_base + t * 128 + (ca & 1) * 64, qd, kd, idesc_qk, 0u, s_full(t, ca & 1));
        ia += a.two ? 1 : 2, ++ca;
        if (ia >= a.j1 - a.j0) mma_commit_elected(q_empty(q_buffer));  // this group's last use of the tile
      }
      if (ca - cb > 1 || !more) {
        if (cb == ca) break;
        while (ib >= b.j1 - b.j0) {
          b_blocks += b.j1 - b.j0;
          walk.next(p, b);
          ib = first_of(b, b_blocks);
        }
        // P V
        const int block = b_blocks + ib, vs = block % TR_V_STAGES, sb = cb & 1;
        ok = wait(v_full(vs), (block / TR_V_STAGES) & 1, TJX_ERR_WAIT_FULL);
        if (ok) ok = wait(p_ready(t, sb), (cb >> 1) & 1, TJX_ERR_WAIT_OTHER);
        if (!ok) break;
        tc_fence_after_sync();
        const uint64_t v0 = smem_desc_sw128(base + L::V_OFF + vs * L::KV_BYTES, L::KV_BYTES / 2, 1024);
        uint64_t vd[4];
        uint32_t pa[4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          vd[kk] = v0 + ((kk * 16 * 128) >> 4);
          pa[kk] = tmem_base + t * 128 + sb * 64 + kk * 8;
        }
        mma_ts_x4_commit(tmem_base + 256 + t * 128, pa, vd, idesc_pv, ib == first_of(b, b_blocks) ? 0u : 1u, o_done(t, sb));
        mma_commit_elected(v_empty(vs));
        ib += b.two ? 1 : 2, ++cb;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and output
    const int t = (warp - 3) >> 2;  // group
    const int quarter = warp & 3;   // TMEM lanes of this warp
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;  // of the tile
    const int node = row / p.group;        // in its tile
    int c = 0, blocks = 0;  // jobs of this group, and blocks of the portions before
    int looked = 0, looked_both = 0, joined = 0;
    bool ok = true;
    auto wait = [&](uint32_t b, uint32_t parity, int code) {
      return tree_wait(b, parity, abort_flag, p.status, code);
    };
    // The product of the group's job c is in the output. A wait tells a barrier's phase from the one before it only, and
    // the scores of job c say that job c - 2 is through, not job c - 1: so even and odd jobs have barriers of their own.
    auto output_done = [&](int c) { return wait(o_done(t, c & 1), (c >> 1) & 1, TJX_ERR_WAIT_OTHER); };
    if (threadIdx.x == 96) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    TreePortion u, next;
    for (bool more = walk.next(p, next); ok && more;) {
      u = next;
      const int n_blocks = u.j1 - u.j0;
      const int tile = u.two ? t : 0;
      const int tile_nodes = u.two ? (tile == 0 ? p.tile_nodes : u.nodes - p.tile_nodes) : u.nodes;
      const int rows = tile_nodes * p.group;
      const bool active = quarter * 32 < rows;  // some row of this warp's is one
      const bool mine_valid = row < rows;
      const int tok = u.tok + tile * p.tile_nodes + node;
      TreeMask mask;
      mask.row = p.tree_mask + static_cast<size_t>(mine_valid ? tok : 0) * p.words, mask.words = mine_valid ? p.words : 0;
      mask.first = mask.words > 0 ? static_cast<uint32_t>(mask.row[0]) : 0u;
      mask.second = mask.words > 1 ? static_cast<uint32_t>(mask.row[1]) : 0u;
      const uint32_t o_tmem = tmem_base + lane_addr + 256 + t * 128;
      float m_used = TR_NOTHING, l = 0.f;
      bool far = false;    // some row's maximum is far from zero
      bool again = false;  // the first loop has left a block to the second, its scores read
      int last_job = -1;
      // Job c: its scores out of TMEM, its weights into it over them. `see0`, `see1`: the positions this row sees, where
      // `masked`. A score that is NaN or plus infinity makes the row NaN, as the formula does: through the maximum, since not
      // every way to an exponential keeps a NaN. Minus infinity weighs nothing beside a larger score and makes a row NaN
      // that has no other (tree_inverse).
      auto job = [&](auto masked, int block, uint32_t see0, uint32_t see1, uint32_t (&pk)[32]) {
        ok = wait(s_full(t, c & 1), (c >> 1) & 1, TJX_ERR_WAIT_TMEM_FULL);
        if (!ok) return;
        tc_fence_after_sync();
        // The scores are there, so the block's keys have been read. (An arrival here is cheaper than the issuer's commit.)
        if (quarter == 0 && lane == 0 && !again) mbar_arrive(k_empty((blocks + block) % TR_K_STAGES));
        if (active) {
          const uint32_t s_tmem = tmem_base + lane_addr + t * 128 + (c & 1) * 64;
          uint32_t v[2][32];
          tmem_ld32(s_tmem, v[0]);
          tmem_ld32(s_tmem + 32, v[1]);
          tmem_wait_ld();
          float m_blk;
          for (bool looked_up = false;; looked_up = true) {
            if (masked.value) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (!((see0 >> i) & 1)) v[0][i] = __float_as_uint(-INFINITY);
                if (!((see1 >> i) & 1)) v[1][i] = __float_as_uint(-INFINITY);
              }
            }
            // (Maxima of two: 64 of them and the exponentials take two warps of a scheduler 830 cycles, 32 maxima of three 1030.)
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 32; ++i) mx[i & 3] = fmax_nan(mx[i & 3], __uint_as_float(v[h][i]));
            m_blk = fmax_nan(fmax_nan(mx[0], mx[1]), fmax_nan(mx[2], mx[3])) * p.scale_log2e;
            if (!masked.value || looked_up || __builtin_expect(!__any_sync(0xFFFFFFFFu, mine_valid && m_blk != m_blk), 1)) break;
            const uint2 paged = tree_paged(p, u.s, (u.j0 + block) * TR_BLOCK);
            see0 &= paged.x, see1 &= paged.y;
          }
          if (m_blk == INFINITY) m_blk = NAN;
          // (Rows of the tile that are none hold other sequences' queries, in place even while those change: they have no say.)
          if (last_job < 0 || __builtin_expect(__any_sync(0xFFFFFFFFu, mine_valid && !(m_blk <= m_used + TR_RESCALE)), 0)) {
            const float m_new = fmax_nan(m_used, m_blk), alpha = ex2(m_used - m_new);
            if (!masked.value && __any_sync(0xFFFFFFFFu, mine_valid && m_blk != m_blk)) {  // (a NaN raises the maximum)
              const uint2 paged = tree_paged(p, u.s, (u.j0 + block) * TR_BLOCK);
              again = (paged.x & paged.y) != 0xFFFFFFFFu;
              if (again) return;
            }
            if (!far && __any_sync(0xFFFFFFFFu, mine_valid && tree_far(m_new))) {
              far = true;
              again = !masked.value;
              if (again) return;
            }
            m_used = m_new;
            if (last_job >= 0) {
              l *= alpha;
              ok = output_done(c - 1);
              tc_fence_after_sync();
#pragma unroll 1
              for (int i = 0; i < 8 && ok; ++i) {
                uint32_t o[16];
                tmem_ld16(o_tmem + i * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                tmem_st16(o_tmem + i * 16, o);
              }
              tmem_wait_st();
            }
          }
          float scale_log2e = p.scale_log2e;
          if (masked.value && __builtin_expect(far, 0)) {
            const bool mine = tree_far(m_used);
            const float factor = mine ? scale_log2e : 1.f;
            scale_log2e = mine ? 1.f : scale_log2e;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 32; ++i) v[h][i] = __float_as_uint(__uint_as_float(v[h][i]) * factor);
          }
          // P is rounded to bf16 for the tensor cores (off by 2^-8 of itself, as in the framework's other attention); the
          // sum adds the unrounded values. Two elements an instruction; a quarter of the exponentials on the FMA pipe, but
          // where positions are hidden: there zero must be zero (a row that sees nothing has the sum 0, one that sees minus
          // infinity only has 1 instead; without hidden positions it has what the FMA pipe's exponentials are held at).
          const float2 scale = make_float2(scale_log2e, scale_log2e), neg_m = make_float2(-m_used, -m_used);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(v[h][i]), __uint_as_float(v[h][i + 1])), scale, neg_m);
              const float2 e = exp2_pair(x, !masked.value && (i & 6) == 6);
              sum[(i >> 1) & 1] = __fadd2_rn(sum[(i >> 1) & 1], e);
              pk[h * 16 + (i >> 1)] = pack_bf16(e.x, e.y);
            }
          l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          if (masked.value && m_used == TR_NOTHING && (see0 | see1) != 0) l = 1.f;
          tmem_st32(s_tmem, pk);
          tmem_wait_st();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(t, c & 1));
        last_job = c;
      };
      int block = u.two ? 0 : (t - blocks) & 1;
      const int step = u.two ? 1 : 2;
      // Blocks that every row sees whole, up to one that has positions without a page, and while no maximum is far from zero
      // (the second loop rounds such scores: 64 products more, whose code in this one would cost more than they do).
      const int plain = min(max(min(u.ctx, u.end) / TR_BLOCK - u.j0, 0), n_blocks);
      for (; block < plain && ok; block += step, ++c) {
        uint32_t pk[32];
        job(std::false_type{}, block, 0u, 0u, pk);
        if (again) break;
      }
      // Blocks with positions that some row does not see, or that are none. What a row does not see must not reach it: zero
      // times NaN is NaN. So rows of V past the end are zeroed, and rows holding anything but finite numbers too, which are
      // then added by hand to the rows that see them. (None of that where the first loop has left a block: its rows are all seen, or
      // zero.)
      for (; block < n_blocks && ok; block += step, ++c) {
        const int kv0 = (u.j0 + block) * TR_BLOCK, stage = (blocks + block) % TR_V_STAGES;
        uint32_t bad[4] = {};
        if (block >= plain) {
          ok = wait(v_full(stage), ((blocks + block) / TR_V_STAGES) & 1, TJX_ERR_WAIT_FULL);
          if (!ok) break;
          const int v_row = row >> 1, limit = u.end - kv0;
          uint4* src = reinterpret_cast<uint4*>(base_ptr + L::V_OFF + stage * L::KV_BYTES + (row & 1) * (L::KV_BYTES / 2) +
                                                v_row * 128);
          __nv_bfloat162 zeros = __floats2bfloat162_rn(0.f, 0.f);
          if (v_row < limit && v_row >= u.ctx - kv0) {  // (what lies before the nodes every row sees)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 x = src[(i + v_row) & 7];  // (eight rows at a time, each at another bank)
              tree_zeros(zeros, x.x), tree_zeros(zeros, x.y), tree_zeros(zeros, x.z), tree_zeros(zeros, x.w);
            }
          }
          const bool odd = __hisnan(zeros.x) || __hisnan(zeros.y);
          uint32_t votes = __ballot_sync(0xFFFFFFFFu, odd);
          votes = (votes | (votes >> 1)) & 0x55555555u;  // bit 2 i: row i of this warp's sixteen
          volatile uint32_t* flags = bad_rows + (t * 2 + (c & 1)) * 4;
          if (lane == 0) {
            flags[quarter] = votes;
            mbar_arrive(u.two ? v_seen_both : v_seen(t));
          }
          ok = u.two ? wait(v_seen_both, looked_both & 1, TJX_ERR_WAIT_OTHER) : wait(v_seen(t), looked & 1, TJX_ERR_WAIT_OTHER);
          if (u.two) ++looked_both; else ++looked;
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 4; ++i) bad[i] = flags[i];
          if (v_row >= limit || ((flags[v_row >> 4] >> (2 * (v_row & 15))) & 1)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) src[(i + v_row) & 7] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        const uint32_t see0 = tree_bits(mask, kv0, u.ctx, u.end), see1 = tree_bits(mask, kv0 + 32, u.ctx, u.end);
        uint32_t pk[32];
        job(std::true_type{}, block, see0, see1, pk);
        again = false;
        if (ok && active && (bad[0] | bad[1] | bad[2] | bad[3]) != 0) {
          // The rows of V that were taken out, once this block's product is in.
          ok = output_done(c);
          if (!ok) break;
          tc_fence_after_sync();
          volatile uint32_t weights_of[32];  // (indexed below: a copy, or P itself would live in local memory in every block)
#pragma unroll
          for (int i = 0; i < 32; ++i) weights_of[i] = pk[i];
#pragma unroll 1
          for (int g = 0; g < TR_BLOCK; ++g) {
            const uint32_t some = g < 32 ? (g < 16 ? bad[0] : bad[1]) : (g < 48 ? bad[2] : bad[3]);
            if (!((some >> (2 * (g & 15))) & 1)) continue;
            const bool sees = ((g < 32 ? see0 : see1) >> (g & 31)) & 1;
            const uint32_t pair = weights_of[g >> 1];
            const float weight = (g & 1) ? bf16_hi(pair) : bf16_lo(pair);
            const int pos = kv0 + g;  // (below the end)
            const int page = min(max(p.page_indices[static_cast<size_t>(u.s) * p.pages_per_seq + pos / p.page_size], 0), p.num_pages - 1);
            const uint32_t* vrow = reinterpret_cast<const uint32_t*>(
                p.kv_cache + (((static_cast<size_t>(page) * p.page_size + pos % p.page_size) * p.Hkv + u.hk) * 2 + 1) * TR_D);
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
              uint32_t o[16];
              tmem_ld16(o_tmem + i * 16, o);
              tmem_wait_ld();
              if (sees) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                  const uint32_t w = vrow[i * 8 + x];
                  o[2 * x] = __float_as_uint(fmaf(weight, bf16_lo(w), __uint_as_float(o[2 * x])));
                  o[2 * x + 1] = __float_as_uint(fmaf(weight, bf16_hi(w), __uint_as_float(o[2 * x + 1])));
                }
              }
              tmem_st16(o_tmem + i * 16, o);
              tmem_wait_st();
            }
          }
          tc_fence_before_sync();
        }
      }
      if (!ok) break;
      more = walk.next(p, next);  // (while the last products run)
      // The portion's end: normalised rows, or a partial result for the join.
      if (last_job >= 0) ok = output_done(last_job);
      if (!ok) break;
      const int part = 2 * blockIdx.x + (u.starts ? 1 : 0);
      const int head = u.hk * p.group + row - node * p.group;
      const size_t part_row = static_cast<size_t>(part) * 32 * p.part_rows + tile * p.tile_nodes * p.group + row;
      // 32 columns from `col` on of every row of the warp (all lanes call it).
      int out_rows[4];  // the rows of the lane's group of four, -1: none
      {
        const int out_row = mine_valid ? tok * p.H + head : -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) out_rows[k] = __shfl_sync(0xFFFFFFFFu, out_row, (lane & ~3) + k);
      }
      auto store32 = [&](int col, const float (&o)[32]) {
        if (u.whole) {
          // Four lanes hold 64 bytes of four rows: they exchange 16-byte pieces, so that a store instruction writes 64
          // bytes of eight rows, not 16 of 32 (each row is a line of its own).
          uint32_t w[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int x = 0; x < 4; ++x) w[k][x] = pack_bf16(o[8 * k + 2 * x], o[8 * k + 2 * x + 1]);
#pragma unroll
          for (int d = 1; d <= 2; d <<= 1)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k & d) continue;
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, (lane & d) ? w[k][x] : w[k + d][x], d);
                if (lane & d) w[k][x] = got; else w[k + d][x] = got;
              }
            }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (out_rows[k] >= 0)
              reinterpret_cast<uint4*>(p.out + static_cast<size_t>(out_rows[k]) * TR_D + col)[lane & 3] =
                  make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        } else if (mine_valid) {
          float4* dst = p.part_o + part_row + static_cast<size_t>(col / 4) * p.part_rows;
#pragma unroll
          for (int x = 0; x < 8; ++x) dst[x * p.part_rows] = make_float4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        }
      };
      const size_t ml_row = static_cast<size_t>(part) * p.part_rows + tile * p.tile_nodes * p.group + row;
      if (u.two) {
        tc_fence_after_sync();
        const float inv = u.whole ? tree_inverse(m_used, l) : 1.0f;
        if (active) {
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            uint32_t o[32];
            tmem_ld32(tmem_base + lane_addr + 256 + t * 128 + i * 32, o);
            tmem_wait_ld();
            float f[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) f[x] = __uint_as_float(o[x]) * inv;
            store32(i * 32, f);
          }
          if (mine_valid && !u.whole) p.part_ml[ml_row] = make_float2(m_used, l);
        }
        tc_fence_before_sync();
      } else {
        // Both groups have a part of the tile's blocks: they exchange their rows' maxima and sums and each joins one
        // half of the columns.
        stats[t * TR_ROWS + row] = make_float2(m_used, l);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(stats_ready);
        ok = wait(stats_ready, joined & 1, TJX_ERR_WAIT_OTHER);
        if (!ok) break;
        tc_fence_after_sync();
        if (active) {
          const float2 a = stats[row], b = stats[TR_ROWS + row];
          const bool has[2] = {n_blocks > ((0 - blocks) & 1), n_blocks > ((1 - blocks) & 1)};  // the group had a block
          const float m = fmaxf(a.x, b.x);
          float w0 = ex2(a.x - m), w1 = ex2(b.x - m);
          const float sum = a.y * w0 + b.y * w1;
          if (u.whole) {
            const float inv = tree_inverse(m, sum);
            w0 *= inv, w1 *= inv;
          }
#pragma unroll 1
          for (int i = 2 * t; i < 2 * t + 2; ++i) {
            uint32_t o0[32], o1[32];
            tmem_ld32(tmem_base + lane_addr + 256 + i * 32, o0);
            tmem_ld32(tmem_base + lane_addr + 384 + i * 32, o1);
            tmem_wait_ld();
            float f[32];
#pragma unroll
            for (int x = 0; x < 32; ++x) {  // (a group without a block has left nothing to read: selected, not weighed)
              f[x] = has[0] ? __uint_as_float(o0[x]) * w0 : 0.f;
              f[x] = has[1] ? fmaf(__uint_as_float(o1[x]), w1, f[x]) : f[x];
            }
            store32(i * 32, f);
          }
          if (mine_valid && !u.whole && t == 0) p.part_ml[ml_row] = make_float2(m, sum);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(outputs_read);
        ok = wait(outputs_read, joined & 1, TJX_ERR_WAIT_OTHER);  // the outputs and the statistics may be overwritten
        ++joined;
        tc_fence_after_sync();
      }
      blocks += n_blocks;
    }
    if (ok && blocks > 0 && u.starts && !u.whole && threadIdx.x == 96)  // (the run's last portion)
      p.joins[blockIdx.x] = make_int4(u.tok, u.nodes, u.hk, static_cast<int>(blockIdx.x + 1 + tree_div(u.past, share)));
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    if (*abort_flag) __nanosleep(100000);
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

constexpr int TJ_WARPS = 8;
constexpr int TJ_BATCH = 4;

// The units that several CTAs shared: a CTA per 32 rows (a lane's) joins their partial results in the order of the
// blocks, a warp 16 of the columns. And the rows that no unit has, which stay the query (CTAs of the first rows only: the
// others' exit would wait for the lengths). Bound by latency, a unit's entry and then its parts: 2.5 us of a call of one
// sequence, 5 of larger ones, of which a launch that returns at once is 0.5 and 0.5 to 1.3.
__global__ void __launch_bounds__(TJ_WARPS * 32) tree_join_kernel(const TreeParams p) {
  int lo = 0, hi = 0;  // the rows that units have (from arrays that were there before either kernel)
  if (blockIdx.y == 0) {
    const int seqs = min(max(p.distribution[0], 0), p.S);
    lo = min(max(p.cu_q_lens[0], 0), p.T), hi = min(max(p.cu_q_lens[seqs], lo), p.T);
  }
  chain_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, x = blockIdx.y * 32 + lane;
  const int4 join = p.joins[blockIdx.x];
  if (x < join.y * p.group) {
    const int first = blockIdx.x, n = join.w - first + 1;  // parts: 2 first + 1, 2 (first + 1), 2 (first + 2), ...
    auto part = [&](int i) { return static_cast<size_t>(2 * (first + i) + (i == 0 ? 1 : 0)); };
    // TJ_BATCH parts' loads at a time, then their turn in order, the running maximum following.
    float m = TR_NOTHING, sum = 0.f, o[16] = {};
    for (int i0 = 0; i0 < n; i0 += TJ_BATCH) {
      float2 ml[TJ_BATCH];
      float4 v[TJ_BATCH][4];
#pragma unroll
      for (int i = 0; i < TJ_BATCH; ++i) {
        if (i0 + i >= n) break;
        ml[i] = p.part_ml[part(i0 + i) * p.part_rows + x];
        const float4* src = p.part_o + (part(i0 + i) * 32 + 4 * warp) * p.part_rows + x;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[i][k] = src[static_cast<size_t>(k) * p.part_rows];
      }
#pragma unroll
      for (int i = 0; i < TJ_BATCH; ++i) {
        if (i0 + i >= n) break;
        const float m_new = fmaxf(m, ml[i].x), a = ex2(m - m_new), w = ex2(ml[i].x - m_new);
        m = m_new;
        sum = fmaf(sum, a, w * ml[i].y);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[4 * k] = fmaf(o[4 * k], a, v[i][k].x * w), o[4 * k + 1] = fmaf(o[4 * k + 1], a, v[i][k].y * w);
          o[4 * k + 2] = fmaf(o[4 * k + 2], a, v[i][k].z * w), o[4 * k + 3] = fmaf(o[4 * k + 3], a, v[i][k].w * w);
        }
      }
    }
    const float inv = tree_inverse(m, sum);
    const size_t row = static_cast<size_t>(join.x + x / p.group) * p.H + join.z * p.group + x % p.group;
    uint4* dst = reinterpret_cast<uint4*>(p.out + row * TR_D + 16 * warp);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      dst[k] = make_uint4(pack_bf16(o[8 * k] * inv, o[8 * k + 1] * inv), pack_bf16(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                          pack_bf16(o[8 * k + 4] * inv, o[8 * k + 5] * inv), pack_bf16(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
  }
  if (blockIdx.y == 0 && p.out != p.q) {
    const size_t units = static_cast<size_t>(p.H) * TR_D / 8;  // 16 bytes each
    const size_t rest = (static_cast<size_t>(lo) + (p.T - hi)) * units;
    const size_t step = static_cast<size_t>(gridDim.x) * TJ_WARPS * 32;
    for (size_t i = static_cast<size_t>(blockIdx.x) * TJ_WARPS * 32 + threadIdx.x; i < rest; i += step) {
      const size_t at = i < lo * units ? i : i + static_cast<size_t>(hi - lo) * units;
      reinterpret_cast<uint4*>(p.out)[at] = reinterpret_cast<const uint4*>(p.q)[at];
    }
  }
}

static size_t tree_align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

static int tree_part_rows(int T, int group) {
  return static_cast<int>(std::min<long long>(2 * TR_ROWS, static_cast<long long>(T) * group));
}

}  // namespace tjx

extern "C" size_t tjx_rpa_tree_attention_workspace_bytes(int T, int S, int H, int Hkv) {
  using namespace tjx;
  if (T <= 0 || S <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0) return 0;
  const size_t ctas = check_device() == 0 ? sm_count() : 148;
  const size_t rows = 2 * ctas * tree_part_rows(T, H / Hkv);
  return tree_align256(ctas * sizeof(int4)) + tree_align256(rows * sizeof(float2)) + tree_align256(rows * TR_D * sizeof(float));
}

extern "C" int tjx_rpa_tree_attention_bf16(const void* q, void* out, const void* kv_cache, const int32_t* kv_lens,
                                           const int32_t* page_indices, const int32_t* cu_q_lens,
                                           const int32_t* tree_mask, const int32_t* distribution, int T, int S, int H,
                                           int Hkv, int D, int words, int page_size, int pages_per_seq, int num_pages,
                                           float sm_scale, void* workspace, size_t workspace_bytes, tjx_stream_t stream) {
  using namespace tjx;
  if (int rc = check_device()) return rc;
  if (!q || !out || !kv_cache || !kv_lens || !page_indices || !cu_q_lens || !tree_mask || !distribution)
    return fail(TJX_E_ARG, "an input or output pointer is null");
  if (T <= 0 || S <= 0 || H <= 0 || Hkv <= 0 || words <= 0 || pages_per_seq <= 0 || num_pages <= 0)
    return fail(TJX_E_ARG, "sizes must be positive");
  if (D != TR_D) return fail(TJX_E_ARG, "head dimension must be 128");
  if (H % Hkv != 0) return fail(TJX_E_ARG, "the query heads must be a multiple of the KV heads");
  if (H / Hkv > TR_ROWS) return fail(TJX_E_LIMIT, "at most 128 query heads per KV head");
  if (page_size <= 0 || page_size % 16 != 0) return fail(TJX_E_ARG, "page_size must be a multiple of 16");
  if (!(sm_scale > 0.f) || sm_scale > 1e30f) return fail(TJX_E_ARG, "sm_scale must be positive");
  if (static_cast<long long>(num_pages) * page_size >= (1ll << 31) || static_cast<long long>(T) * H >= (1ll << 31) ||
      static_cast<long long>(S) * pages_per_seq >= (1ll << 31) ||
      static_cast<long long>(pages_per_seq) * page_size >= (1ll << 31) - TR_BLOCK)
    return fail(TJX_E_LIMIT, "num_pages * page_size, pages_per_seq * page_size, S * pages_per_seq and T * H must fit in int32");
  for (const void* ptr : {q, static_cast<const void*>(out), kv_cache})
    if (reinterpret_cast<uintptr_t>(ptr) & 15u) return fail(TJX_E_ARG, "q, out and kv_cache must be 16-byte aligned");
  const size_t need = tjx_rpa_tree_attention_workspace_bytes(T, S, H, Hkv);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(TJX_E_ARG, "workspace is null or smaller than tjx_rpa_tree_attention_workspace_bytes");
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return fail(TJX_E_ARG, "workspace must be 256-byte aligned");
  TreeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q), p.out = static_cast<__nv_bfloat16*>(out);
  p.kv_cache = static_cast<const __nv_bfloat16*>(kv_cache);
  p.kv_lens = kv_lens, p.page_indices = page_indices, p.cu_q_lens = cu_q_lens, p.tree_mask = tree_mask;
  p.distribution = distribution;
  p.T = T, p.S = S, p.H = H, p.Hkv = Hkv, p.group = H / Hkv, p.page_size = page_size, p.pages_per_seq = pages_per_seq;
  p.num_pages = num_pages, p.words = words, p.scale_log2e = sm_scale * TR_LOG2E;
  p.tile_nodes = TR_ROWS / p.group;
  p.box_rows = std::min(page_size & -page_size, TR_BLOCK);
  p.status = device_status_word();
  if (p.status == nullptr) return fail(TJX_E_CUDA, "could not locate the device status word");
  const int ctas = sm_count();
  p.per_cta = 1.0 / ctas;
  p.part_rows = tree_part_rows(T, p.group);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  p.joins = reinterpret_cast<int4*>(w), w += tree_align256(ctas * sizeof(int4));
  p.part_ml = reinterpret_cast<float2*>(w), w += tree_align256(2ull * ctas * p.part_rows * sizeof(float2));
  p.part_o = reinterpret_cast<float4*>(w);

  CUtensorMap mq, mk, mv;
  {
    const uint64_t dims[3] = {TR_D, static_cast<uint64_t>(H), static_cast<uint64_t>(T)};
    const uint64_t strides[2] = {TR_D * 2, static_cast<uint64_t>(H) * TR_D * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.tile_nodes)};
    if (int rc = make_tensor_map(&mq, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
  }
  {
    const uint64_t dims[3] = {TR_D, static_cast<uint64_t>(Hkv) * 2, static_cast<uint64_t>(num_pages) * page_size};
    const uint64_t strides[2] = {TR_D * 2, static_cast<uint64_t>(Hkv) * 2 * TR_D * 2};
    const uint32_t box[3] = {64, 1, static_cast<uint32_t>(p.box_rows)};
    if (int rc = make_tensor_map(&mk, kv_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NAN_REQUEST_ZERO_FMA))
      return rc;
    if (int rc = make_tensor_map(&mv, kv_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return rc;
  }
  static bool configured[64] = {};
  int dev = 0;
  TJX_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    TJX_CUDA(cudaFuncSetAttribute(tree_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TreeSmem::TOTAL));
    configured[dev & 63] = true;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  tree_kernel<<<ctas, TR_THREADS, TreeSmem::TOTAL, s>>>(mq, mk, mv, p);
  TJX_CUDA(cudaGetLastError());
  TJX_CUDA(launch_chained(tree_join_kernel, dim3(ctas, (p.part_rows + 31) / 32), dim3(TJ_WARPS * 32), 0, s, p));
  return 0;
}
