// What a step on the ragged paged cache (examples/ragged_paged_attention.py: pages of page_size positions, each
// position's heads with key and value side by side) needs around its attention, made on the device from the requests'
// lengths and the projection's output:
//   rpa_plan_kernel        block tables, slot map, positions and token offsets of the step from the requests' lengths
//   norm_rope_kernel       RMS norm of every query and key head and its rotation by the token's position; keys and
//                          values straight into their cache rows
//   rpa_commit_kernel      the rows of an accepted path of drafted tokens moved behind the cached prefix
#include <algorithm>

#include "tjx_host.cuh"
#include "tjx_ptx.cuh"

#include "../../include/tilejax_b200.h"

namespace tjx {

// ------------------------------------------------------------------------------------------ block tables and slots

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_SEQS = 8192;  // 16 bytes of shared memory each

struct PlanParams {
  const int32_t *ctx_lens, *q_lens, *held, *depths;  // held, depths: or null
  int32_t* page_indices;
  const int32_t *free_pages, *n_free;
  int free_capacity;
  int S, T, pages_per_seq, page_size;
  int32_t *kv_lens, *cu_q_lens, *positions, *slots, *held_out, *n_free_out;
};

// A sequence as the scan leaves it in shared memory.
struct PlanSeq {
  int first, lack;  // its first token (clipped to T), its first fresh page
  int ctx, held;
};

// Inclusive sums over the CTA's threads, and the sums of all of them. `sums` is not reused before a __syncthreads.
struct PlanSums {
  long long q[32];
  int n[32];
};
__device__ __forceinline__ void plan_scan(PlanSums& sums, long long& q, int& n, long long& all_q, int& all_n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long yq = __shfl_up_sync(0xFFFFFFFFu, q, d);
    const int yn = __shfl_up_sync(0xFFFFFFFFu, n, d);
    if (lane >= d) q += yq, n += yn;
  }
  if (lane == 31) sums.q[warp] = q, sums.n[warp] = n;
  __syncthreads();
  long long wq = sums.q[lane];  // every warp adds the warps' sums up for itself
  int wn = sums.n[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long yq = __shfl_up_sync(0xFFFFFFFFu, wq, d);
    const int yn = __shfl_up_sync(0xFFFFFFFFu, wn, d);
    if (lane >= d) wq += yq, wn += yn;
  }
  all_q = __shfl_sync(0xFFFFFFFFu, wq, 31), all_n = __shfl_sync(0xFFFFFFFFu, wn, 31);
  const long long bq = __shfl_sync(0xFFFFFFFFu, wq, max(warp - 1, 0));
  const int bn = __shfl_sync(0xFFFFFFFFu, wn, max(warp - 1, 0));
  if (warp > 0) q += bq, n += bn;
}

// Every CTA scans all sequences (new tokens, and pages a sequence lacks) into shared memory and then takes its share of
// the tokens and of the pages handed out; CTA 0 also writes what there is one of per sequence. Nothing a CTA reads is
// written by another: table entries below a sequence's held pages are only read, those handed out only written (a token on
// such a page takes it from the free list itself). Bound by latency: a load, a scan, a search and a load more.
__global__ void __launch_bounds__(PLAN_THREADS, 2) rpa_plan_kernel(const PlanParams p) {
  extern __shared__ __align__(16) uint8_t plan_smem[];
  PlanSeq* seq = reinterpret_cast<PlanSeq*>(plan_smem);  // [S + 1], the last: all tokens, all fresh pages
  __shared__ PlanSums sums[2];
  const int t = threadIdx.x;
  const int free_now = min(max(p.n_free[0], 0), p.free_capacity);
  auto lacking = [&](int ctx, int held, long long tokens) {
    const long long len = min(static_cast<long long>(ctx) + tokens, 0x7FFFFFFFll);
    const unsigned pages = (static_cast<unsigned>(len) + static_cast<unsigned>(p.page_size) - 1u) / static_cast<unsigned>(p.page_size);
    return max(static_cast<int>(min(pages, static_cast<unsigned>(p.pages_per_seq))) - held, 0);
  };
  long long tokens = 0;  // of the sequences before
  int fresh_pages = 0;
  for (int s0 = 0, round = 0; s0 < p.S; s0 += PLAN_THREADS, ++round) {
    const int s = s0 + t;
    PlanSeq me{0, 0, 0, 0};
    long long q = 0;
    int n = 0;
    if (s < p.S) {
      me.ctx = max(p.ctx_lens[s], 0), q = max(p.q_lens[s], 0);
      const unsigned cached = (static_cast<unsigned>(me.ctx) + static_cast<unsigned>(p.page_size) - 1u) / static_cast<unsigned>(p.page_size);
      const int held = p.held != nullptr ? p.held[s] : static_cast<int>(min(cached, static_cast<unsigned>(p.pages_per_seq)));
      me.held = min(max(held, 0), p.pages_per_seq);
      n = lacking(me.ctx, me.held, q);
    }
    long long upto_q = q, all_q;
    int upto_n = n, all_n;
    plan_scan(sums[round & 1], upto_q, upto_n, all_q, all_n);
    me.first = static_cast<int>(min(tokens + upto_q - q, static_cast<long long>(p.T)));
    me.lack = fresh_pages + upto_n - n;
    if (s < p.S) seq[s] = me;
    tokens += all_q, fresh_pages += all_n;
  }
  const int total = static_cast<int>(min(tokens, static_cast<long long>(p.T)));
  if (t == 0) seq[p.S] = PlanSeq{total, fresh_pages, 0, 0};
  __syncthreads();
  if (tokens > p.T) {  // rows for some of the tokens only: the pages again, for those
    fresh_pages = 0;
    for (int s0 = 0, round = 0; s0 < p.S; s0 += PLAN_THREADS, ++round) {
      const int s = s0 + t;
      long long q = 0, all_q;
      int n = s < p.S ? lacking(seq[s].ctx, seq[s].held, seq[s + 1].first - seq[s].first) : 0, all_n;
      int upto_n = n;
      __syncthreads();
      plan_scan(sums[round & 1], q, upto_n, all_q, all_n);
      if (s < p.S) seq[s].lack = fresh_pages + upto_n - n;
      fresh_pages += all_n;
    }
    if (t == 0) seq[p.S].lack = fresh_pages;
    __syncthreads();
  }
  if (blockIdx.x == 0) {
    for (int s = t; s < p.S; s += PLAN_THREADS) {
      const PlanSeq me = seq[s];
      const int lacks = seq[s + 1].lack - me.lack;
      p.kv_lens[s] = static_cast<int>(min(static_cast<long long>(me.ctx) + (seq[s + 1].first - me.first), 0x7FFFFFFFll));
      p.cu_q_lens[s] = me.first;
      p.held_out[s] = me.held + min(max(free_now - me.lack, 0), lacks);
    }
    if (t == 0) {
      p.cu_q_lens[p.S] = total;
      p.n_free_out[0] = max(free_now - fresh_pages, 0);
      p.n_free_out[1] = max(fresh_pages - free_now, 0);
    }
  }
  const int step = static_cast<int>(gridDim.x) * PLAN_THREADS, me = static_cast<int>(blockIdx.x) * PLAN_THREADS + t;
  // The last sequence that starts at or before x, by its first token or its first fresh page.
  auto find = [&](auto key, int x) {
    int lo = 0, hi = p.S + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (key(seq[mid]) <= x) lo = mid; else hi = mid;
    }
    return lo;
  };
  // The k-th page handed out comes off the top of the free stack, or is missing.
  auto fresh = [&](int k) { return k < free_now ? p.free_pages[free_now - 1 - k] : -1; };
  for (int k = me; k < fresh_pages; k += step) {
    const int s = find([](const PlanSeq& x) { return x.lack; }, k);
    p.page_indices[static_cast<size_t>(s) * p.pages_per_seq + seq[s].held + (k - seq[s].lack)] = fresh(k);
  }
  for (int i = me; i < p.T; i += step) {
    int position = 0, slot = -1;
    if (i < total) {
      const int s = find([](const PlanSeq& x) { return x.first; }, i);
      const PlanSeq of = seq[s];
      const unsigned place = static_cast<unsigned>(of.ctx) + static_cast<unsigned>(i - of.first);
      const unsigned page = place / static_cast<unsigned>(p.page_size), row = place - page * static_cast<unsigned>(p.page_size);
      position = p.depths != nullptr ? of.ctx + p.depths[i] : static_cast<int>(place);
      if (page < static_cast<unsigned>(p.pages_per_seq)) {
        const int entry = static_cast<int>(page) < of.held
                              ? p.page_indices[static_cast<size_t>(s) * p.pages_per_seq + page]
                              : fresh(of.lack + static_cast<int>(page) - of.held);
        const long long at = static_cast<long long>(entry) * p.page_size + row;
        if (entry >= 0 && at <= 0x7FFFFFFFll) slot = static_cast<int>(at);  // (a table's entry may be anything)
      }
    }
    p.positions[i] = position;
    p.slots[i] = slot;
  }
}

// ------------------------------------------------------------------------------------------ norm, rotation, write

constexpr int NR_THREADS = 256;
constexpr int NR_UNROLL = 4;
constexpr int NR_BLOCKS = 2;  // CTAs of an SM. Fewer or more of them, or of rows in flight, are slower: 4096 tokens of 32 + 8
                              // + 8 heads 21.5 us; 30 with one CTA, 29 with three; 24 with two, five or six rows a lane

struct NormRopeParams {
  const __nv_bfloat16 *q, *k, *v;                // v: or null (no cache)
  const __nv_bfloat16 *q_gamma, *k_gamma;        // [D], or both null
  __nv_bfloat16 *q_out, *k_out, *kv_cache;       // k_out or kv_cache
  long long q_tok, k_tok, v_tok, qo_tok, ko_tok;  // elements from one token to the next
  long long q_head, k_head, v_head, qo_head, ko_head;  // ... and from one head to the next
  const int32_t *positions, *slots;
  const float* cos_sin;  // [max_positions, rot]: cosines, then sines
  int T, H, Hkv, rot, max_positions, n_slots;
  bool wide;  // every row starts at a multiple of 16 bytes (else of 8)
  float eps;
};

// D / 8 lanes make a row; a lane holds eight elements of it as four pairs that rotate together: 4 u .. 4 u + 3 of lane u,
// which are 16 neighbouring bytes where pairs are neighbours (NEIGHBOURS), else two runs of four, one in each half of the
// rotated part; lanes past it hold elements that are only normed. So the rotation needs no exchange between lanes. With
// (a, b) a pair, g its gammas and r = 1 / rms:  r (a g_a cos - b g_b sin),  r (a g_a sin + b g_b cos), the four products of
// gamma and angle made once for all heads of the token, everything f32 from the load to the one rounding of the result.
//
// Heads come in chunks of one kind (queries, keys, values), NR_UNROLL rows a lane. The chunks of all tokens, in order, are
// cut into equal runs, one for each warp the GPU holds at a time (a single token's chunks each get a warp), and a warp has
// the next chunk's rows, and the next token's angles, on their way while it works on one. Each row is read once and written
// once; beside the memory the issue of instructions bounds it: 130 for two rows of 128 (issue slots 60 % busy) where
// unfolded factors, one element an instruction and shuffles between the halves took 200 (77 %). 4096 tokens of 32 + 8 + 8
// heads 21.5 us, 16384 76 us; 16384 of 32 + 8 without a cache 63 us: 5.6 to 5.9 TB/s behind 3 to 5 us that do not depend on
// the size. (Loads past the L1, or to be dropped first: as
// fast or a tenth slower.)
template <int D, bool NEIGHBOURS>
__global__ void __launch_bounds__(NR_THREADS, NR_BLOCKS) norm_rope_kernel(const NormRopeParams p) {
  constexpr int LANES = D / 8;            // lanes per row
  constexpr int PER_PASS = 32 / LANES;    // rows per warp and pass
  constexpr int ROWS = PER_PASS * NR_UNROLL;
  const int lane = threadIdx.x & 31, u = lane % LANES, sub = lane / LANES;
  const int chunks_q = (p.H + ROWS - 1) / ROWS, chunks_k = (p.Hkv + ROWS - 1) / ROWS;
  const int chunks = chunks_q + (p.v != nullptr ? 2 : 1) * chunks_k;
  const long long total = static_cast<long long>(p.T) * chunks, warps = static_cast<long long>(gridDim.x) * (NR_THREADS / 32);
  const long long warp = static_cast<long long>(blockIdx.x) * (NR_THREADS / 32) + (threadIdx.x >> 5);
  const long long run = warp * total / warps, run_end = (warp + 1) * total / warps;
  if (run >= run_end) return;
  int tok = static_cast<int>(run / chunks), chunk = static_cast<int>(run % chunks);
  const bool rotated = u < p.rot / 8;
  // The lane's elements: a .. a + 3 and b .. b + 3.
  const int a = !NEIGHBOURS && rotated ? 4 * u : 8 * u;
  const int b = !NEIGHBOURS && rotated ? p.rot / 2 + 4 * u : a + 4;
  const bool wide = NEIGHBOURS && p.wide;
  auto load = [&](const __nv_bfloat16* src) {
    if (wide) return *reinterpret_cast<const uint4*>(src + a);
    const uint2 lo = *reinterpret_cast<const uint2*>(src + a), hi = *reinterpret_cast<const uint2*>(src + b);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  // Kind of a chunk (0 queries, 1 keys, 2 values) and its first head.
  auto kind_of = [&](int chunk) { return chunk < chunks_q ? 0 : chunk < chunks_q + chunks_k ? 1 : 2; };
  auto head_of = [&](int chunk, int kind) { return (chunk - (kind == 0 ? 0 : kind == 1 ? chunks_q : chunks_q + chunks_k)) * ROWS; };
  auto load_chunk = [&](int tok, int chunk, uint4 (&x)[NR_UNROLL]) {
    const int kind = kind_of(chunk), r0 = head_of(chunk, kind) + sub;
    const __nv_bfloat16* src = kind == 0 ? p.q + tok * p.q_tok : kind == 1 ? p.k + tok * p.k_tok : p.v + tok * p.v_tok;
    const long long head = kind == 0 ? p.q_head : kind == 1 ? p.k_head : p.v_head;
    const int heads = kind == 0 ? p.H : p.Hkv;
#pragma unroll
    for (int i = 0; i < NR_UNROLL; ++i) {
      const int r = r0 + i * PER_PASS;
      x[i] = r < heads ? load(src + r * head) : make_uint4(0, 0, 0, 0);
    }
  };
  // Pairs j = 2 h and 2 h + 1 of a lane's words, first and second elements.
  auto unpack = [](const uint4& w, float2 (&fa)[2], float2 (&fb)[2]) {
    if (NEIGHBOURS) {
      fa[0] = make_float2(bf16_lo(w.x), bf16_lo(w.y)), fb[0] = make_float2(bf16_hi(w.x), bf16_hi(w.y));
      fa[1] = make_float2(bf16_lo(w.z), bf16_lo(w.w)), fb[1] = make_float2(bf16_hi(w.z), bf16_hi(w.w));
    } else {
      fa[0] = make_float2(bf16_lo(w.x), bf16_hi(w.x)), fa[1] = make_float2(bf16_lo(w.y), bf16_hi(w.y));
      fb[0] = make_float2(bf16_lo(w.z), bf16_hi(w.z)), fb[1] = make_float2(bf16_lo(w.w), bf16_hi(w.w));
    }
  };
  // A token's angles: of its position, clamped to the table as a gather's index is.
  auto load_angles = [&](int position, float4& cs, float4& sn) {
    cs = make_float4(1.f, 1.f, 1.f, 1.f), sn = make_float4(0.f, 0.f, 0.f, 0.f);
    if (!rotated) return;
    const float* table = p.cos_sin + static_cast<size_t>(min(max(position, 0), p.max_positions - 1)) * p.rot + 4 * u;
    cs = *reinterpret_cast<const float4*>(table), sn = *reinterpret_cast<const float4*>(table + p.rot / 2);
  };
  uint4 x[NR_UNROLL];
  load_chunk(tok, chunk, x);
  float4 cs, sn;
  load_angles(p.positions[tok], cs, sn);
  int slot = p.slots != nullptr ? p.slots[tok] : -1;
  int position_ahead = tok + 1 < p.T ? p.positions[tok + 1] : 0;
  int slot_ahead = p.slots != nullptr && tok + 1 < p.T ? p.slots[tok + 1] : -1;
  int have = -1;  // the kind the factors are of
  float2 aa[2], ab[2], ba[2], bb[2];  // first = a aa + b ab, second = a ba + b bb
  for (long long at = run; at < run_end; ++at) {
    uint4 ahead[NR_UNROLL];
    float4 cs_ahead = cs, sn_ahead = sn;
    const bool new_token = chunk + 1 == chunks;
    if (at + 1 < run_end) {
      load_chunk(new_token ? tok + 1 : tok, new_token ? 0 : chunk + 1, ahead);
      if (new_token) load_angles(position_ahead, cs_ahead, sn_ahead);
    }
    const int kind = kind_of(chunk), r0 = head_of(chunk, kind) + sub;
    if (kind != have && kind < 2) {
      have = kind;
      float2 ga[2] = {make_float2(1.f, 1.f), make_float2(1.f, 1.f)}, gb[2] = {ga[0], ga[0]};
      if (p.q_gamma != nullptr) unpack(load(kind == 0 ? p.q_gamma : p.k_gamma), ga, gb);
      const float2 c[2] = {make_float2(cs.x, cs.y), make_float2(cs.z, cs.w)}, s[2] = {make_float2(sn.x, sn.y), make_float2(sn.z, sn.w)};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        aa[h] = __fmul2_rn(ga[h], c[h]), bb[h] = __fmul2_rn(gb[h], c[h]), ba[h] = __fmul2_rn(ga[h], s[h]);
        ab[h] = __fmul2_rn(gb[h], make_float2(-s[h].x, -s[h].y));
      }
    }
    __nv_bfloat16* dst = nullptr;
    long long head = 0;
    if (kind == 0)
      dst = p.q_out + tok * p.qo_tok, head = p.qo_head;
    else if (p.kv_cache == nullptr)
      dst = p.k_out + tok * p.ko_tok, head = p.ko_head;
    else if (slot >= 0 && slot < p.n_slots)
      dst = p.kv_cache + (static_cast<size_t>(slot) * p.Hkv * 2 + (kind - 1)) * D, head = 2 * D;
    const int heads = dst == nullptr ? 0 : kind == 0 ? p.H : p.Hkv;
#pragma unroll
    for (int i = 0; i < NR_UNROLL; ++i) {
      uint4 y = x[i];
      if (kind < 2) {
        float2 fa[2], fb[2];
        unpack(y, fa, fb);
        float scale = 1.f;
        if (p.q_gamma != nullptr) {
          float2 sum = __fmul2_rn(fa[0], fa[0]);
          sum = __ffma2_rn(fa[1], fa[1], sum), sum = __ffma2_rn(fb[0], fb[0], sum), sum = __ffma2_rn(fb[1], fb[1], sum);
          float squares = sum.x + sum.y;
#pragma unroll
          for (int d = LANES / 2; d >= 1; d >>= 1) squares += __shfl_xor_sync(0xFFFFFFFFu, squares, d);
          scale = rsqrtf(fmaf(squares, 1.0f / D, p.eps));
        }
        const float2 sc = make_float2(scale, scale);
        float2 ya[2], yb[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (rotated) {
            ya[h] = __ffma2_rn(fa[h], aa[h], __fmul2_rn(fb[h], ab[h]));
            yb[h] = __ffma2_rn(fa[h], ba[h], __fmul2_rn(fb[h], bb[h]));
          } else {  // (an infinity must not meet a sine of 0)
            ya[h] = __fmul2_rn(fa[h], aa[h]), yb[h] = __fmul2_rn(fb[h], bb[h]);
          }
          ya[h] = __fmul2_rn(ya[h], sc), yb[h] = __fmul2_rn(yb[h], sc);
        }
        y = NEIGHBOURS ? make_uint4(pack_bf16(ya[0].x, yb[0].x), pack_bf16(ya[0].y, yb[0].y), pack_bf16(ya[1].x, yb[1].x),
                                    pack_bf16(ya[1].y, yb[1].y))
                       : make_uint4(pack_bf16(ya[0].x, ya[0].y), pack_bf16(ya[1].x, ya[1].y), pack_bf16(yb[0].x, yb[0].y),
                                    pack_bf16(yb[1].x, yb[1].y));
      }
      const int r = r0 + i * PER_PASS;
      if (r < heads) {
        __nv_bfloat16* to = dst + r * head;
        if (wide) {
          *reinterpret_cast<uint4*>(to + a) = y;
        } else {
          *reinterpret_cast<uint2*>(to + a) = make_uint2(y.x, y.y);
          *reinterpret_cast<uint2*>(to + b) = make_uint2(y.z, y.w);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NR_UNROLL; ++i) x[i] = ahead[i];
    ++chunk;
    if (new_token) {
      chunk = 0, ++tok, have = -1;
      cs = cs_ahead, sn = sn_ahead, slot = slot_ahead;
      if (tok + 1 < p.T) {
        position_ahead = p.positions[tok + 1];
        if (p.slots != nullptr) slot_ahead = p.slots[tok + 1];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ accepted path

constexpr int COMMIT_THREADS = 256;
constexpr int COMMIT_BATCH = 16;

// A CTA moves one sequence's accepted rows, each thread a 16-byte column of them, in path order and COMMIT_BATCH rows at a
// time: a warp looks the batch's entries up (a lane each), then all loads of the batch come before its stores. The path's
// nodes ascend, so node d's row never lies in front of row d, no batch overwrites a row a later batch reads, and columns
// are independent. Bound by latency: lengths, path, table and rows, one after the other. (With every thread looking every
// entry up, its two divisions by the page size each, 256 sequences took 9.7 us.)
__global__ void __launch_bounds__(COMMIT_THREADS)
    rpa_commit_kernel(uint4* __restrict__ kv_cache, const int32_t* __restrict__ kv_lens,
                      const int32_t* __restrict__ page_indices, const int32_t* __restrict__ cu_q_lens,
                      const int32_t* __restrict__ paths, const int32_t* __restrict__ n_accepted, int P, int row_units,
                      int page_size, int pages_per_seq, int num_pages, int32_t* __restrict__ out_lens) {
  __shared__ long long from_sh[COMMIT_BATCH], to_sh[COMMIT_BATCH];
  __shared__ int count_sh;
  const int s = blockIdx.x, col = blockIdx.y * COMMIT_THREADS + threadIdx.x;
  const int kv_len = kv_lens[s], q_len = max(cu_q_lens[s + 1] - cu_q_lens[s], 0), asked = n_accepted[s];
  if (asked < 0) {  // nothing was drafted: every new token stays
    if (col == 0) out_lens[s] = kv_len;
    return;
  }
  const int ctx = max(kv_len - q_len, 0), limit = min(asked, P);
  const int32_t* path = paths + static_cast<size_t>(s) * P;
  const int32_t* table = page_indices + static_cast<size_t>(s) * pages_per_seq;
  auto row = [&](int place) -> long long {  // 16-byte units from the cache's start, or -1: no such row
    const int entry = place / page_size;
    if (place < 0 || entry >= pages_per_seq) return -1;
    const int page = table[entry];
    if (page < 0 || page >= num_pages) return -1;
    return (static_cast<long long>(page) * page_size + (place - entry * page_size)) * row_units;
  };
  int kept = 0, last = -1;  // (last: of the looking warp)
  for (int d0 = 0; d0 < limit; d0 += COMMIT_BATCH) {
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x, d = d0 + lane;
      const bool here = lane < COMMIT_BATCH && d < limit;
      const int node = here ? path[d] : -1;
      const int before = __shfl_up_sync(0xFFFFFFFFu, node, 1);
      // The path ends in front of the first entry that does not ascend or is no new token.
      const uint32_t wrong = __ballot_sync(0xFFFFFFFFu, !here || node <= (lane == 0 ? last : before) || node >= q_len);
      const int count = wrong == 0 ? 32 : __ffs(wrong) - 1;
      if (lane < count) {
        const bool moves = node != d;  // (else it is where it belongs)
        const long long from = moves ? row(ctx + node) : -1, to = moves ? row(ctx + d) : -1;
        from_sh[lane] = from, to_sh[lane] = from < 0 ? -1 : to;
      }
      if (lane == 0) count_sh = count;
      last = __shfl_sync(0xFFFFFFFFu, node, max(count - 1, 0));
    }
    __syncthreads();
    const int count = count_sh;
    if (col < row_units) {
      uint4 data[COMMIT_BATCH];
#pragma unroll
      for (int i = 0; i < COMMIT_BATCH; ++i)
        if (i < count && to_sh[i] >= 0) data[i] = kv_cache[from_sh[i] + col];
#pragma unroll
      for (int i = 0; i < COMMIT_BATCH; ++i)
        if (i < count && to_sh[i] >= 0) kv_cache[to_sh[i] + col] = data[i];
    }
    kept += count;
    __syncthreads();
    if (count < min(limit - d0, COMMIT_BATCH)) break;
  }
  if (col == 0) out_lens[s] = ctx + kept;
}

}  // namespace tjx

extern "C" {

int tjx_rpa_plan(const int32_t* ctx_lens, const int32_t* q_lens, const int32_t* pages_held, const int32_t* depths,
                 int32_t* page_indices, const int32_t* free_pages, const int32_t* n_free, int free_capacity, int S, int T,
                 int pages_per_seq, int page_size, int32_t* kv_lens, int32_t* cu_q_lens, int32_t* positions,
                 int32_t* slots, int32_t* pages_held_out, int32_t* n_free_out, tjx_stream_t stream) {
  using namespace tjx;
  if (int rc = check_device()) return rc;
  if (!ctx_lens || !q_lens || !page_indices || !n_free || !kv_lens || !cu_q_lens || !pages_held_out || !n_free_out ||
      (T > 0 && (!positions || !slots)) || (free_capacity > 0 && !free_pages))
    return fail(TJX_E_ARG, "an input or output pointer is null");
  if (S <= 0 || T < 0 || pages_per_seq <= 0 || page_size <= 0 || free_capacity < 0)
    return fail(TJX_E_ARG, "sizes must be positive");
  if (S > PLAN_MAX_SEQS) return fail(TJX_E_LIMIT, "more than 8192 sequences");
  if (static_cast<long long>(S) * pages_per_seq >= (1ll << 31))
    return fail(TJX_E_LIMIT, "S * pages_per_seq must fit in int32");
  if (T > (1 << 30)) return fail(TJX_E_LIMIT, "more than 2^30 tokens");
  PlanParams p{};
  p.ctx_lens = ctx_lens, p.q_lens = q_lens, p.held = pages_held, p.depths = depths;
  p.page_indices = page_indices, p.free_pages = free_pages, p.n_free = n_free, p.free_capacity = free_capacity;
  p.S = S, p.T = T, p.pages_per_seq = pages_per_seq, p.page_size = page_size;
  p.kv_lens = kv_lens, p.cu_q_lens = cu_q_lens, p.positions = positions, p.slots = slots;
  p.held_out = pages_held_out, p.n_free_out = n_free_out;
  const size_t smem = static_cast<size_t>(S + 1) * sizeof(PlanSeq);
  static bool configured[64] = {};
  int dev = 0;
  TJX_CUDA(cudaGetDevice(&dev));
  if (!configured[dev & 63]) {
    TJX_CUDA(cudaFuncSetAttribute(rpa_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>((PLAN_MAX_SEQS + 1) * sizeof(PlanSeq))));
    configured[dev & 63] = true;
  }
  const int grid = std::max(1, std::min((T + PLAN_THREADS - 1) / PLAN_THREADS, 2 * sm_count()));
  rpa_plan_kernel<<<grid, PLAN_THREADS, smem, static_cast<cudaStream_t>(stream)>>>(p);
  TJX_CUDA(cudaGetLastError());
  return 0;
}

int tjx_norm_rope_bf16(const void* q, const void* k, const void* v, const int64_t* strides, const void* q_gamma,
                       const void* k_gamma, const int32_t* positions, const float* cos_sin, const int32_t* slots,
                       void* q_out, void* k_out, void* kv_cache, int T, int H, int Hkv, int D, int rot, int max_positions,
                       int interleaved, int n_slots, float eps, tjx_stream_t stream) {
  using namespace tjx;
  if (int rc = check_device()) return rc;
  if (!q || !k || !strides || !positions || (rot > 0 && !cos_sin) || !q_out) return fail(TJX_E_ARG, "an input or output pointer is null");
  if ((q_gamma == nullptr) != (k_gamma == nullptr)) return fail(TJX_E_ARG, "q_gamma and k_gamma are given together or not at all");
  const bool to_cache = kv_cache != nullptr;
  if (to_cache ? (!v || !slots || n_slots <= 0) : (!k_out || v != nullptr || slots != nullptr))
    return fail(TJX_E_ARG, "v, slots and kv_cache go together, or k_out alone");
  if (T <= 0 || H <= 0 || Hkv <= 0 || max_positions <= 0) return fail(TJX_E_ARG, "sizes must be positive");
  if (D != 64 && D != 128 && D != 256) return fail(TJX_E_ARG, "head dimension must be 64, 128 or 256");
  if (rot < 0 || rot > D || rot % 8 != 0) return fail(TJX_E_ARG, "the rotated part is a multiple of 8, at most the head dimension");
  if (!(eps >= 0.f)) return fail(TJX_E_ARG, "eps must not be negative");
  // 16 bytes a lane where every row allows it.
  uintptr_t bits = 0;
  for (const void* ptr : {q, k, v, q_gamma, k_gamma, const_cast<const void*>(q_out), const_cast<const void*>(k_out), const_cast<const void*>(kv_cache)})
    bits |= reinterpret_cast<uintptr_t>(ptr);
  if (bits & 7u) return fail(TJX_E_ARG, "bf16 operands must be 8-byte aligned");
  if (reinterpret_cast<uintptr_t>(cos_sin) & 15u) return fail(TJX_E_ARG, "cos_sin must be 16-byte aligned");
  for (int i = 0; i < 10; ++i) {
    if (strides[i] % 4 != 0 || strides[i] < 0) return fail(TJX_E_ARG, "strides must be multiples of 4 elements");
    bits |= static_cast<uintptr_t>(strides[i]) * 2;
  }
  const bool wide = (bits & 15u) == 0;
  NormRopeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q), p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.q_gamma = static_cast<const __nv_bfloat16*>(q_gamma), p.k_gamma = static_cast<const __nv_bfloat16*>(k_gamma);
  p.q_out = static_cast<__nv_bfloat16*>(q_out), p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.kv_cache = static_cast<__nv_bfloat16*>(kv_cache);
  p.q_tok = strides[0], p.q_head = strides[1], p.k_tok = strides[2], p.k_head = strides[3], p.v_tok = strides[4];
  p.v_head = strides[5], p.qo_tok = strides[6], p.qo_head = strides[7], p.ko_tok = strides[8], p.ko_head = strides[9];
  p.positions = positions, p.slots = slots, p.cos_sin = cos_sin;
  p.T = T, p.H = H, p.Hkv = Hkv, p.rot = rot, p.max_positions = max_positions, p.wide = wide;
  p.n_slots = n_slots, p.eps = eps;
  const int rows = NR_UNROLL * 32 / (D / 8);
  const int chunks = (H + rows - 1) / rows + (to_cache ? 2 : 1) * ((Hkv + rows - 1) / rows);
  const long long blocks = (static_cast<long long>(T) * chunks + NR_THREADS / 32 - 1) / (NR_THREADS / 32);
  const int grid = static_cast<int>(std::min<long long>(blocks, sm_count() * NR_BLOCKS));
  auto kernel = interleaved ? (D == 64 ? norm_rope_kernel<64, true> : D == 128 ? norm_rope_kernel<128, true> : norm_rope_kernel<256, true>)
                            : (D == 64 ? norm_rope_kernel<64, false> : D == 128 ? norm_rope_kernel<128, false> : norm_rope_kernel<256, false>);
  kernel<<<grid, NR_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(p);
  TJX_CUDA(cudaGetLastError());
  return 0;
}

int tjx_rpa_commit_bf16(void* kv_cache, const int32_t* kv_lens, const int32_t* page_indices, const int32_t* cu_q_lens,
                        const int32_t* paths, const int32_t* n_accepted, int32_t* out_lens, int S, int P, int Hkv, int D,
                        int page_size, int pages_per_seq, int num_pages, tjx_stream_t stream) {
  using namespace tjx;
  if (int rc = check_device()) return rc;
  if (!kv_cache || !kv_lens || !page_indices || !cu_q_lens || !paths || !n_accepted || !out_lens)
    return fail(TJX_E_ARG, "an input or output pointer is null");
  if (S <= 0 || P <= 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || pages_per_seq <= 0 || num_pages <= 0)
    return fail(TJX_E_ARG, "sizes must be positive");
  if (D % 8 != 0) return fail(TJX_E_ARG, "head dimension must be a multiple of 8");
  if (reinterpret_cast<uintptr_t>(kv_cache) & 15u) return fail(TJX_E_ARG, "kv_cache must be 16-byte aligned");
  if (static_cast<long long>(Hkv) * D > (1ll << 24)) return fail(TJX_E_LIMIT, "Hkv * D is too large");
  const int row_units = Hkv * 2 * D * 2 / 16;
  const dim3 grid(S, (row_units + COMMIT_THREADS - 1) / COMMIT_THREADS);
  rpa_commit_kernel<<<grid, COMMIT_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<uint4*>(kv_cache), kv_lens, page_indices, cu_q_lens, paths, n_accepted, P, row_units, page_size,
      pages_per_seq, num_pages, out_lens);
  TJX_CUDA(cudaGetLastError());
  return 0;
}

}  // extern "C"
