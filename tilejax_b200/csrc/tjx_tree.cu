// Attention of a tree of drafted tokens over the ragged paged cache: the decode case of ragged paged attention
// (examples/ragged_paged_attention.py:121-149) for sequences that bring several tokens of which each sees the cached
// prefix and those of its own sequence that its mask names (its ancestors in the tree, and itself).
//   o[t, h] = sum_p softmax_p(sm_scale q[t, h] . k[p, h / group]) v[p, h / group]
// over the positions p < kv_len - q_len and the nodes j (position kv_len - q_len + j) with bit j of tree_mask[t] set.
#include <algorithm>

#include "tjx_host.cuh"
#include "tjx_ptx.cuh"

#include "../../include/tilejax_b200.h"

namespace tjx {

constexpr int TR_D = 128;
constexpr float TR_LOG2E = 1.4426950408889634f;

struct TreeParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const __nv_bfloat16* kv_cache;
  const int32_t *kv_lens, *page_indices, *cu_q_lens, *tree_mask, *distribution;
  int T, S, H, Hkv, group, page_size, pages_per_seq, num_pages, words;
  float scale_log2e;
};

// A warp per (token, query head): 32 positions at a time, a lane per position for the scores (q in shared memory, the
// lane reads its key's row), then four of the 128 output dimensions per lane. Positions the mask hides are skipped, so
// what they hold does not matter.
__global__ void __launch_bounds__(128) tree_simple_kernel(const TreeParams p) {
  __shared__ float q_sh[4][TR_D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (item >= static_cast<long long>(p.T) * p.H) return;
  const int t = static_cast<int>(item / p.H), h = static_cast<int>(item % p.H), hk = h / p.group;
  const uint2 raw = reinterpret_cast<const uint2*>(p.q + item * TR_D)[lane];
  const int seqs = min(max(p.distribution[0], 0), p.S);
  int lo = 0, hi = seqs;  // the sequence of token t: cu_q_lens[lo] <= t < cu_q_lens[lo + 1]
  const bool covered = seqs > 0 && t >= p.cu_q_lens[0] && t < p.cu_q_lens[seqs];
  uint2* dst = reinterpret_cast<uint2*>(p.out + item * TR_D) + lane;
  if (!covered) {
    if (p.out != p.q) *dst = raw;
    return;
  }
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q_lens[mid] <= t) lo = mid; else hi = mid;
  }
  const int s = lo, q_len = p.cu_q_lens[s + 1] - p.cu_q_lens[s];
  const long long ctx = static_cast<long long>(p.kv_lens[s]) - q_len;
  const int end = static_cast<int>(min(static_cast<long long>(max(p.kv_lens[s], 0)),
                                       static_cast<long long>(p.pages_per_seq) * p.page_size));
  q_sh[warp][4 * lane] = bf16_lo(raw.x) * p.scale_log2e, q_sh[warp][4 * lane + 1] = bf16_hi(raw.x) * p.scale_log2e;
  q_sh[warp][4 * lane + 2] = bf16_lo(raw.y) * p.scale_log2e, q_sh[warp][4 * lane + 3] = bf16_hi(raw.y) * p.scale_log2e;
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < end; p0 += 32) {
    const int pos = p0 + lane;
    bool sees = pos < end;
    if (sees && pos >= ctx) {
      const long long node = pos - ctx;
      sees = node < 32ll * p.words && ((p.tree_mask[static_cast<size_t>(t) * p.words + node / 32] >> (node % 32)) & 1);
    }
    float score = 0.f;
    long long row = 0;
    if (pos < end) {
      const int page = min(max(p.page_indices[static_cast<size_t>(s) * p.pages_per_seq + pos / p.page_size], 0), p.num_pages - 1);
      row = ((static_cast<long long>(page) * p.page_size + pos % p.page_size) * p.Hkv + hk) * 2 * TR_D;
    }
    if (sees) {
      const uint4* k = reinterpret_cast<const uint4*>(p.kv_cache + row);
#pragma unroll 4
      for (int u = 0; u < TR_D / 8; ++u) {
        const uint4 x = k[u];
        const float* qv = &q_sh[warp][8 * u];
        score += qv[0] * bf16_lo(x.x) + qv[1] * bf16_hi(x.x) + qv[2] * bf16_lo(x.y) + qv[3] * bf16_hi(x.y) +
                 qv[4] * bf16_lo(x.z) + qv[5] * bf16_hi(x.z) + qv[6] * bf16_lo(x.w) + qv[7] * bf16_hi(x.w);
      }
    }
    const unsigned seen = __ballot_sync(0xFFFFFFFFu, sees);
    if (seen == 0) continue;
    float mx = sees ? score : -INFINITY;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
    const float m_new = fmaxf(m, mx), alpha = ex2(m - m_new);
    const float e = sees ? ex2(score - m_new) : 0.f;
    m = m_new;
    float sum = e;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    l = l * alpha + sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= alpha;
    for (int i = 0; i < 32; ++i) {
      const float w = __shfl_sync(0xFFFFFFFFu, e, i);
      const long long r = __shfl_sync(0xFFFFFFFFu, row, i);
      if (!((seen >> i) & 1)) continue;
      const uint2 v = reinterpret_cast<const uint2*>(p.kv_cache + r + TR_D)[lane];
      o[0] += w * bf16_lo(v.x), o[1] += w * bf16_hi(v.x), o[2] += w * bf16_lo(v.y), o[3] += w * bf16_hi(v.y);
    }
  }
  const float inv = m == -INFINITY ? 0.f : 1.f / l;  // a row that sees nothing is zero
  *dst = make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

}  // namespace tjx

extern "C" size_t tjx_rpa_tree_attention_workspace_bytes(int T, int S, int H, int Hkv) {
  if (T <= 0 || S <= 0 || H <= 0 || Hkv <= 0) return 0;
  return 256;
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
  if (H / Hkv > 128) return fail(TJX_E_LIMIT, "at most 128 query heads per KV head");
  if (page_size <= 0 || page_size % 16 != 0) return fail(TJX_E_ARG, "page_size must be a multiple of 16");
  if (!(sm_scale > 0.f) || sm_scale > 1e30f) return fail(TJX_E_ARG, "sm_scale must be positive");
  if (static_cast<long long>(num_pages) * page_size >= (1ll << 31) || static_cast<long long>(T) * H >= (1ll << 31) ||
      static_cast<long long>(S) * pages_per_seq >= (1ll << 31) || static_cast<long long>(pages_per_seq) * page_size >= (1ll << 31))
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
  const long long warps = static_cast<long long>(T) * H;
  tree_simple_kernel<<<static_cast<unsigned>((warps + 3) / 4), 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
  TJX_CUDA(cudaGetLastError());
  return 0;
}
