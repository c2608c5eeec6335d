// Eviction from a KV cache by accumulated attention weight on B200 (sm_100a).
//
// Each (layer, trace, KV head) keeps `budget` of its len rows: those whose position is
// recent (>= next_pos - recent) or among the first `sinks`, then the rows of largest
// score, ties to the lowest row. Attention does not depend on the order of a cache's
// rows, so nothing is shifted: the j-th row at or beyond the budget that stays (a mover)
// goes into the j-th row below the budget that leaves (a hole). Holes and movers are
// disjoint, so the moves have no order among them; only moved rows cost bandwidth.
#include <algorithm>

#include "common.cuh"

namespace mb {

struct EvictArgs {
  uint16_t *k, *v;
  int64_t ks[4], vs[4];  // element strides (layer, trace, head, row)
  const float* scores;
  const int32_t* positions;
  float* scores_out;
  int32_t* positions_out;
  const int32_t *lens, *next_pos;
  int32_t* lens_out;
  int32_t* moves;  // [units][2][cap]: holes, movers
  int64_t cap;
  int layers, T, Hkv, Lmax, d, budget, recent, sinks, vec;
};

constexpr int kEvictBlock = 1024;

// Order-preserving image of a row's rank: a guarded row above everything, NaN below
// everything, -0 equal to +0.
__device__ __forceinline__ uint32_t rank_code(float s, bool guarded) {
  if (guarded) return 0xFFFFFFFFu;
  if (s != s) return 0u;
  const uint32_t b = __float_as_uint(s + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ bool guarded_row(int pos, int64_t recent_from, int sinks) {
  return pos >= recent_from || pos < sinks;
}

// Exclusive prefix of a 0/1 flag over the block, and the block's total.
__device__ __forceinline__ int block_rank(bool flag, int* wsum, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const uint32_t b = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) wsum[w] = __popc(b);
  __syncthreads();
  int before = 0, all = 0;
  for (int u = 0; u < kEvictBlock / 32; ++u) {
    const int c = wsum[u];
    before += u < w ? c : 0;
    all += c;
  }
  __syncthreads();
  *total = all;
  return before + __popc(b & ((1u << lane) - 1));
}

// One CTA per (layer, trace, KV head).
__global__ void __launch_bounds__(kEvictBlock) k_evict(EvictArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ int wsum[kEvictBlock / 32];
  __shared__ uint32_t prefix_s;
  __shared__ int need_s;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int64_t unit = blockIdx.x;
  const int h = unit % a.Hkv, t = (unit / a.Hkv) % a.T, layer = unit / (static_cast<int64_t>(a.Hkv) * a.T);
  const int len = max(0, min(a.lens[t], a.Lmax));
  const int kept = min(len, a.budget);
  const int64_t recent_from = static_cast<int64_t>(a.next_pos[t]) - a.recent;
  const float* sc = a.scores + unit * a.Lmax;
  const int32_t* ps = a.positions + unit * a.Lmax;
  float* so = a.scores_out + unit * a.Lmax;
  int32_t* po = a.positions_out + unit * a.Lmax;
  if (h == 0 && layer == 0 && tid == 0) a.lens_out[t] = kept;
  if (len == kept) {  // nothing leaves
    if (so != sc)
      for (int r = tid; r < len; r += kEvictBlock) {
        so[r] = sc[r];
        po[r] = ps[r];
      }
    return;
  }
  // the kept-th largest code, eight bits at a time, and how many rows of exactly that code stay
  uint32_t prefix = 0;
  int need = kept;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int r = tid; r < len; r += kEvictBlock) {
      const uint32_t c = rank_code(sc[r], guarded_row(ps[r], recent_from, a.sinks));
      if (shift == 24 || (c >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(c >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int left = need, b = 255;
      while (b > 0 && static_cast<int>(hist[b]) < left) left -= hist[b--];
      prefix_s = prefix | (static_cast<uint32_t>(b) << shift);
      need_s = left;
    }
    __syncthreads();
    prefix = prefix_s;
    need = need_s;
  }
  // in row order: which rows of the threshold code stay, the holes and the movers
  int32_t* holes = a.moves + unit * 2 * a.cap;
  int32_t* movers = holes + a.cap;
  int ties = 0, nh = 0, nm = 0, all;
  for (int r0 = 0; r0 < len; r0 += kEvictBlock) {
    const int r = r0 + tid;
    const uint32_t c = r < len ? rank_code(sc[r], guarded_row(ps[r], recent_from, a.sinks)) : 0u;
    const bool tie = r < len && c == prefix;
    const int before = block_rank(tie, wsum, &all);
    const bool stays = r < len && (c > prefix || (tie && ties + before < need));
    ties += all;
    const bool hole = r < kept && !stays, mover = r >= kept && stays;
    const int hr = block_rank(hole, wsum, &all);
    if (hole) holes[nh + hr] = r;
    nh += all;
    const int mr = block_rank(mover, wsum, &all);
    if (mover) movers[nm + mr] = r;
    nm += all;
    if (stays && r < kept && so != sc) {
      so[r] = sc[r];
      po[r] = ps[r];
    }
  }
  __syncthreads();
  const int n = min(nh, nm);  // equal: as many rows leave below the budget as stay beyond it
  for (int j = tid; j < n; j += kEvictBlock) {
    so[holes[j]] = sc[movers[j]];
    po[holes[j]] = ps[movers[j]];
  }
  uint16_t* k = a.k + layer * a.ks[0] + t * a.ks[1] + h * a.ks[2];
  uint16_t* v = a.v + layer * a.vs[0] + t * a.vs[1] + h * a.vs[2];
  if (a.vec) {
    const int per = a.d / 8;
    for (int64_t e = tid; e < static_cast<int64_t>(n) * per; e += kEvictBlock) {
      const int j = e / per, c = (e - static_cast<int64_t>(j) * per) * 8;
      *reinterpret_cast<uint4*>(k + holes[j] * a.ks[3] + c) =
          *reinterpret_cast<const uint4*>(k + movers[j] * a.ks[3] + c);
      *reinterpret_cast<uint4*>(v + holes[j] * a.vs[3] + c) =
          *reinterpret_cast<const uint4*>(v + movers[j] * a.vs[3] + c);
    }
  } else {
    for (int64_t e = tid; e < static_cast<int64_t>(n) * a.d; e += kEvictBlock) {
      const int j = e / a.d, c = e - static_cast<int64_t>(j) * a.d;
      k[holes[j] * a.ks[3] + c] = k[movers[j] * a.ks[3] + c];
      v[holes[j] * a.vs[3] + c] = v[movers[j] * a.vs[3] + c];
    }
  }
}

}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_cache_evict_workspace_size(int32_t layers, int32_t T, int32_t Hkv, int32_t Lmax, int32_t budget) {
  if (layers < 1 || T < 1 || Hkv < 1 || Lmax < 1 || budget < 1) return 0;
  const size_t cap = budget < Lmax ? std::min(budget, Lmax - budget) : 0;
  return (static_cast<size_t>(layers) * T * Hkv * 2 * cap * 4 + 255) / 256 * 256 + 256;
}

int32_t mb_cache_evict(uint16_t* k_cache, uint16_t* v_cache, const int64_t* strides, const float* scores,
                       const int32_t* positions, float* scores_out, int32_t* positions_out, const int32_t* lens,
                       const int32_t* next_pos, int32_t* lens_out, int32_t layers, int32_t T, int32_t Hkv,
                       int32_t Lmax, int32_t d, int32_t budget, int32_t recent, int32_t sinks, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (!k_cache || !v_cache || !strides || !scores || !positions || !scores_out || !positions_out || !lens ||
      !next_pos || !lens_out)
    return MB_ERR_NULL;
  if (layers < 1 || T < 1 || Hkv < 1 || Lmax < 1 || d < 1 || budget < 1 || recent < 0 || sinks < 0) return MB_ERR_ARGS;
  if (static_cast<int64_t>(recent) + sinks > budget) return MB_ERR_ARGS;
  if (lens_out == lens) return MB_ERR_ARGS;  // every CTA reads the old lengths
  if ((scores_out == scores) != (positions_out == positions)) return MB_ERR_ARGS;
  const int64_t units = static_cast<int64_t>(layers) * T * Hkv;
  if (units > 0x7FFFFFFFll || Lmax > 0x7FFF0000) return MB_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < mb_cache_evict_workspace_size(layers, T, Hkv, Lmax, budget))
    return MB_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return MB_ERR_ALIGN;
  EvictArgs a;
  a.k = k_cache;
  a.v = v_cache;
  bool vec = d % 8 == 0 && aligned(k_cache, 16) && aligned(v_cache, 16);
  for (int u = 0; u < 4; ++u) {
    a.ks[u] = strides[u];
    a.vs[u] = strides[4 + u];
  }
  for (int u = 0; u < 8; ++u) vec = vec && strides[u] % 8 == 0;
  a.vec = vec;
  a.scores = scores;
  a.positions = positions;
  a.scores_out = scores_out;
  a.positions_out = positions_out;
  a.lens = lens;
  a.next_pos = next_pos;
  a.lens_out = lens_out;
  a.moves = static_cast<int32_t*>(workspace);
  a.cap = budget < Lmax ? std::min(budget, Lmax - budget) : 0;
  a.layers = layers;
  a.T = T;
  a.Hkv = Hkv;
  a.Lmax = Lmax;
  a.d = d;
  a.budget = budget;
  a.recent = recent;
  a.sinks = sinks;
  return launch_with_pdl(k_evict, dim3(static_cast<unsigned>(units)), dim3(kEvictBlock), 0,
                         static_cast<cudaStream_t>(stream), a);
}

}  // extern "C"
