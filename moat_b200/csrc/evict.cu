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
  int32_t* moves;   // [units][2][cap]: holes, movers (two-kernel form)
  int32_t* counts;  // [units] (two-kernel form)
  int cap, slice;   // most moves of a unit; most rows of a CTA
  int layers, T, Hkv, Lmax, d, budget, recent, sinks;
  bool vec, vec_ranks;  // 16-byte pieces of rows; of scores and positions
};

constexpr int kMaxWarps = 32;

// Order-preserving image of a row's rank: a guarded row above everything, NaN below
// everything, -0 equal to +0.
__device__ __forceinline__ uint32_t rank_code(float s, int pos, int64_t recent_from, int sinks) {
  if (pos >= recent_from || pos < sinks) return 0xFFFFFFFFu;
  if (s != s) return 0u;
  const uint32_t b = __float_as_uint(s + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Moves row `from` to row `to` of both caches, `per` 16-byte pieces each; the thread does the
// pieces of moves first, first + step, ... of n, four moves' loads in flight.
__device__ __forceinline__ void move_rows(const EvictArgs& a, uint16_t* k, uint16_t* v, const int32_t* holes,
                                          const int32_t* movers, int n, int tid, int threads) {
  if (a.vec) {
    const int per = a.d / 8, group = threads / per;  // moves done side by side
    const int first = tid / per, c = (tid - first * per) * 8;
    if (first >= group) return;
    constexpr int kU = 4;
    for (int j0 = first; j0 < n; j0 += kU * group) {
      uint4 x[kU], y[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int j = j0 + u * group;
        if (j < n) {
          const int64_t from = movers[j];
          x[u] = *reinterpret_cast<const uint4*>(k + from * a.ks[3] + c);
          y[u] = *reinterpret_cast<const uint4*>(v + from * a.vs[3] + c);
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int j = j0 + u * group;
        if (j < n) {
          const int64_t to = holes[j];
          *reinterpret_cast<uint4*>(k + to * a.ks[3] + c) = x[u];
          *reinterpret_cast<uint4*>(v + to * a.vs[3] + c) = y[u];
        }
      }
    }
  } else {
    for (int64_t e = tid; e < static_cast<int64_t>(n) * a.d; e += threads) {
      const int j = static_cast<int>(e / a.d), c = static_cast<int>(e - static_cast<int64_t>(j) * a.d);
      const int64_t from = movers[j], to = holes[j];
      k[to * a.ks[3] + c] = k[from * a.ks[3] + c];
      v[to * a.vs[3] + c] = v[from * a.vs[3] + c];
    }
  }
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int CS>
__device__ __forceinline__ void unit_sync() {
  if (CS > 1)
    cluster_sync();
  else
    __syncthreads();
}

// Sum over the cluster's lower ranks of *word (same place in every CTA), and over all of them.
template <int CS>
__device__ __forceinline__ int ranks_before(uint32_t* word, uint32_t rank, int* all) {
  if (CS == 1) {
    *all = static_cast<int>(*word);
    return 0;
  }
  int before = 0, total = 0;
#pragma unroll
  for (uint32_t r = 0; r < CS; ++r) {
    const int v = static_cast<int>(ld_cluster_u32(mapa_shared(smem_u32(word), r)));
    before += r < rank ? v : 0;
    total += v;
  }
  *all = total;
  return before;
}

// Selection for one (layer, trace, KV head) by a cluster of CS CTAs, each with a slice of the
// rows. The ranks stay in shared memory: scores and positions are read once. The kept-th
// largest rank is found eight bits at a time from histograms (joined through distributed
// shared memory); then every warp sweeps its own run of rows, so that ties, holes and movers
// are numbered in row order with one exchange of counts each. FUSED (CS = 1): the same CTA
// moves the rows; otherwise the numbered moves go to the workspace for k_evict_move.
template <int CS, bool FUSED>
__global__ void __launch_bounds__(1024) k_evict(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t dyn[];
  __shared__ uint32_t hist[256];  // this CTA's
  __shared__ uint32_t digit_s, need_s;
  __shared__ uint32_t wties[kMaxWarps + 1], wholes[kMaxWarps + 1], wmovers[kMaxWarps + 1];  // [kMaxWarps]: the CTA's
  uint32_t* code = dyn;               // [slice]
  uint32_t* stay = code + a.slice;    // [slice / 32]
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const uint32_t rank = CS > 1 ? cluster_ctarank() : 0;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t unit = blockIdx.x / CS;
  const int h = unit % a.Hkv, t = (unit / a.Hkv) % a.T, layer = unit / (static_cast<int64_t>(a.Hkv) * a.T);
  const int len = max(0, min(a.lens[t], a.Lmax));
  const int kept = min(len, a.budget);
  const int64_t recent_from = static_cast<int64_t>(a.next_pos[t]) - a.recent;
  const float* sc = a.scores + unit * a.Lmax;
  const int32_t* ps = a.positions + unit * a.Lmax;
  float* so = a.scores_out + unit * a.Lmax;
  int32_t* po = a.positions_out + unit * a.Lmax;
  // this CTA's rows [r0, r0 + n), the same share of the valid rows for every CTA
  const int share = ((len + CS - 1) / CS + 127) & ~127;
  const int r0 = min(len, static_cast<int>(rank) * share), n = min(share, len - r0);
  if (h == 0 && layer == 0 && rank == 0 && tid == 0) a.lens_out[t] = kept;
  if (len == kept) {  // nothing leaves
    if (!FUSED && rank == 0 && tid == 0) a.counts[unit] = 0;
    if (so != sc)
      for (int i = tid; i < n; i += threads) {
        so[r0 + i] = sc[r0 + i];
        po[r0 + i] = ps[r0 + i];
      }
    return;  // the whole cluster
  }
  // ranks, and the histogram of their first digit
  for (int i = tid; i < 256; i += threads) hist[i] = 0;
  __syncthreads();
  if (a.vec_ranks) {  // r0 is a multiple of 128
    const float4* s4 = reinterpret_cast<const float4*>(sc + r0);
    const int4* p4 = reinterpret_cast<const int4*>(ps + r0);
#pragma unroll 4
    for (int i = tid; i < (n + 3) / 4; i += threads) {
      const float4 s = s4[i];  // may read past len, never past Lmax
      const int4 p = p4[i];
      const uint4 c = make_uint4(rank_code(s.x, p.x, recent_from, a.sinks), rank_code(s.y, p.y, recent_from, a.sinks),
                                 rank_code(s.z, p.z, recent_from, a.sinks), rank_code(s.w, p.w, recent_from, a.sinks));
      *reinterpret_cast<uint4*>(code + 4 * i) = c;
      if (4 * i < n) atomicAdd(&hist[c.x >> 24], 1u);
      if (4 * i + 1 < n) atomicAdd(&hist[c.y >> 24], 1u);
      if (4 * i + 2 < n) atomicAdd(&hist[c.z >> 24], 1u);
      if (4 * i + 3 < n) atomicAdd(&hist[c.w >> 24], 1u);
    }
  } else {
#pragma unroll 4
    for (int i = tid; i < n; i += threads) {
      const uint32_t c = rank_code(sc[r0 + i], ps[r0 + i], recent_from, a.sinks);
      code[i] = c;
      atomicAdd(&hist[c >> 24], 1u);
    }
  }
  uint32_t prefix = 0;
  int need = kept;
  for (int shift = 24;; shift -= 8) {
    unit_sync<CS>();
    if (warp == 0) {  // lane l has digits 255 - 8 l downwards; find the digit where the count reaches need
      uint32_t bin[8];
      int sum = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int b = 255 - 8 * lane - u;
        if (CS == 1) {
          bin[u] = hist[b];
        } else {
          bin[u] = 0;
#pragma unroll
          for (uint32_t r = 0; r < CS; ++r) bin[u] += ld_cluster_u32(mapa_shared(smem_u32(&hist[b]), r));
        }
        sum += bin[u];
      }
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
      }
      const int first = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;  // need <= rows: one lane has it
      if (lane == first) {
        int left = need - (upto - sum), u = 0;
        while (u < 7 && static_cast<int>(bin[u]) < left) left -= bin[u++];
        digit_s = 255 - 8 * lane - u;
        need_s = left;
      }
    }
    unit_sync<CS>();  // also: every CTA has read the histograms
    prefix |= digit_s << shift;
    need = need_s;
    if (shift == 0) break;
    for (int i = tid; i < 256; i += threads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += threads) {
      const uint32_t c = code[i];
      if ((c >> shift) == (prefix >> shift)) atomicAdd(&hist[(c >> (shift - 8)) & 255], 1u);
    }
  }
  // every warp's run of rows, whole words of 32
  const int words = (n + 31) / 32, per = (words + warps - 1) / warps;
  const int w0 = min(words, warp * per), w1 = min(words, w0 + per);
  int ties = 0;
  for (int w = w0; w < w1; ++w) {
    const int i = w * 32 + lane;
    ties += __popc(__ballot_sync(0xffffffffu, i < n && code[i] == prefix));
  }
  auto number = [&](uint32_t* counts, int mine) {  // this warp's first number among the unit's, counts[kMaxWarps] the CTA's
    if (lane == 0) counts[warp] = mine;
    __syncthreads();
    if (warp == 0) {
      const int v = lane < warps ? static_cast<int>(counts[lane]) : 0;
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      counts[lane] = x - v;
      if (lane == 31) counts[kMaxWarps] = x;
    }
  };
  number(wties, ties);
  unit_sync<CS>();
  int all;
  int tie = ranks_before<CS>(&wties[kMaxWarps], rank, &all) + wties[warp];
  int holes = 0, movers = 0;
  for (int w = w0; w < w1; ++w) {  // the first `need` ties stay
    const int i = w * 32 + lane;
    const uint32_t c = i < n ? code[i] : 0u;
    const uint32_t tied = __ballot_sync(0xffffffffu, i < n && c == prefix);
    const bool stays = i < n && (c > prefix || (c == prefix && tie + __popc(tied & ((1u << lane) - 1)) < need));
    tie += __popc(tied);
    const uint32_t bits = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) stay[w] = bits;
    const uint32_t low = __ballot_sync(0xffffffffu, i < n && r0 + i < kept);
    holes += __popc(low & ~bits);
    movers += __popc(bits & ~low);
  }
  number(wholes, holes);
  number(wmovers, movers);
  unit_sync<CS>();
  int n_moves;
  int hole = ranks_before<CS>(&wholes[kMaxWarps], rank, &all) + wholes[warp];
  int mover = ranks_before<CS>(&wmovers[kMaxWarps], rank, &n_moves) + wmovers[warp];
  // as many rows leave below the budget as stay beyond it
  int32_t* hole_list = FUSED ? reinterpret_cast<int32_t*>(stay + a.slice / 32) : a.moves + unit * 2 * a.cap;
  int32_t* mover_list = hole_list + a.cap;
  for (int w = w0; w < w1; ++w) {
    const int r = r0 + w * 32 + lane;
    const uint32_t bits = stay[w], low = __ballot_sync(0xffffffffu, r < kept);
    const uint32_t valid = __ballot_sync(0xffffffffu, r < r0 + n), below = (1u << lane) - 1;
    const uint32_t hb = valid & low & ~bits, mb = bits & ~low;
    if ((hb >> lane) & 1) hole_list[hole + __popc(hb & below)] = r;
    if ((mb >> lane) & 1) mover_list[mover + __popc(mb & below)] = r;
    hole += __popc(hb);
    mover += __popc(mb);
    if (so != sc && ((bits & low) >> lane) & 1) {
      so[r] = sc[r];
      po[r] = ps[r];
    }
  }
  if (CS > 1) unit_sync<CS>();  // no CTA leaves while others read its counts
  if (!FUSED) {
    if (rank == 0 && tid == 0) a.counts[unit] = n_moves;
    return;
  }
  __syncthreads();
  for (int j = tid; j < n_moves; j += threads) {
    so[hole_list[j]] = sc[mover_list[j]];
    po[hole_list[j]] = ps[mover_list[j]];
  }
  move_rows(a, a.k + layer * a.ks[0] + t * a.ks[1] + h * a.ks[2], a.v + layer * a.vs[0] + t * a.vs[1] + h * a.vs[2],
            hole_list, mover_list, n_moves, tid, threads);
}

// The moves of the two-kernel form: CTA (x, y) does moves x * kMoveChunk ... of unit unit0 + y.
constexpr int kMoveThreads = 256;
constexpr int kMoveChunk = 128;

__global__ void __launch_bounds__(kMoveThreads) k_evict_move(const __grid_constant__ EvictArgs a, int64_t unit0) {
  pdl_wait();
  pdl_launch_dependents();
  const int64_t unit = unit0 + blockIdx.y;
  const int first = blockIdx.x * kMoveChunk, n = min(kMoveChunk, a.counts[unit] - first);
  if (n <= 0) return;
  const int h = unit % a.Hkv, t = (unit / a.Hkv) % a.T, layer = unit / (static_cast<int64_t>(a.Hkv) * a.T);
  const int32_t* holes = a.moves + unit * 2 * a.cap + first;
  const int32_t* movers = holes + a.cap;
  const int64_t base = unit * a.Lmax;
  for (int j = threadIdx.x; j < n; j += kMoveThreads) {
    a.scores_out[base + holes[j]] = a.scores[base + movers[j]];
    a.positions_out[base + holes[j]] = a.positions[base + movers[j]];
  }
  move_rows(a, a.k + layer * a.ks[0] + t * a.ks[1] + h * a.ks[2], a.v + layer * a.vs[0] + t * a.vs[1] + h * a.vs[2],
            holes, movers, n, threadIdx.x, kMoveThreads);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct EvictPlan {
  int cs, threads, slice, cap;
  bool fused;
  size_t smem;
};

constexpr int kMaxSlice = 48 * 1024;  // ranks of a CTA: 192 KB

static bool evict_plan(int64_t units, int Lmax, int d, int budget, EvictPlan* pl) {
  pl->cap = budget < Lmax ? std::min(budget, Lmax - budget) : 0;
  // One CTA that also moves its rows, where the units alone fill the GPU or the moves are few
  // (a second kernel costs more than the moves); its lists lie in shared memory.
  pl->fused = Lmax <= 4096 && (units >= 2 * sm_count() || static_cast<int64_t>(pl->cap) * d <= 32 * 1024);
  pl->cs = 1;
  if (!pl->fused)  // enough CTAs per unit to use the SMs, slices that fit
    while (pl->cs < 16 && ((Lmax + pl->cs - 1) / pl->cs > kMaxSlice ||
                          (pl->cs < 8 && units * pl->cs * 2 <= sm_count() && Lmax / pl->cs > 2048)))
      pl->cs *= 2;
  pl->slice = ((Lmax + pl->cs - 1) / pl->cs + 127) & ~127;
  if (pl->slice > kMaxSlice) return false;
  pl->threads = pl->slice <= 1024 ? 256 : pl->slice <= 4096 ? 512 : 1024;
  pl->smem = static_cast<size_t>(pl->slice) * 4 + pl->slice / 8 + (pl->fused ? static_cast<size_t>(pl->cap) * 8 : 0);
  return true;
}

template <int CS, bool FUSED>
static int launch_select(const EvictArgs& a, const EvictPlan& pl, int64_t units, cudaStream_t st) {
  auto kern = k_evict<CS, FUSED>;
  if (pl.smem > 40 * 1024 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024) != cudaSuccess) {
    (void)cudaGetLastError();
    return MB_ERR_LAUNCH;
  }
  if (CS > 8 && cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    (void)cudaGetLastError();
    return MB_ERR_LAUNCH;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units * CS));
  cfg.blockDim = dim3(pl.threads);
  cfg.dynamicSmemBytes = pl.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CS > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) {
    (void)cudaGetLastError();
    return MB_ERR_LAUNCH;
  }
  return MB_OK;
}

}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_cache_evict_workspace_size(int32_t layers, int32_t T, int32_t Hkv, int32_t Lmax, int32_t budget) {
  if (layers < 1 || T < 1 || Hkv < 1 || Lmax < 1 || budget < 1) return 0;
  const size_t cap = budget < Lmax ? std::min(budget, Lmax - budget) : 0;
  return static_cast<size_t>(layers) * T * Hkv * (2 * cap + 1) * 4 + 256;
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
  EvictPlan pl;
  if (units > 0x7FFFFFFll || !evict_plan(units, Lmax, d, budget, &pl)) return MB_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < mb_cache_evict_workspace_size(layers, T, Hkv, Lmax, budget))
    return MB_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return MB_ERR_ALIGN;
  EvictArgs a;
  a.k = k_cache;
  a.v = v_cache;
  bool vec = d % 8 == 0 && d <= 1024 && aligned(k_cache, 16) && aligned(v_cache, 16);
  for (int u = 0; u < 4; ++u) {
    a.ks[u] = strides[u];
    a.vs[u] = strides[4 + u];
  }
  for (int u = 0; u < 8; ++u) vec = vec && strides[u] % 8 == 0;
  a.vec = vec;
  a.vec_ranks = Lmax % 4 == 0 && aligned(scores, 16) && aligned(positions, 16);
  a.scores = scores;
  a.positions = positions;
  a.scores_out = scores_out;
  a.positions_out = positions_out;
  a.lens = lens;
  a.next_pos = next_pos;
  a.lens_out = lens_out;
  a.counts = static_cast<int32_t*>(workspace);
  a.moves = a.counts + units;
  a.cap = pl.cap;
  a.slice = pl.slice;
  a.layers = layers;
  a.T = T;
  a.Hkv = Hkv;
  a.Lmax = Lmax;
  a.d = d;
  a.budget = budget;
  a.recent = recent;
  a.sinks = sinks;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pl.fused) return launch_select<1, true>(a, pl, units, st);
  const int rc = pl.cs == 1   ? launch_select<1, false>(a, pl, units, st)
                 : pl.cs == 2 ? launch_select<2, false>(a, pl, units, st)
                 : pl.cs == 4 ? launch_select<4, false>(a, pl, units, st)
                 : pl.cs == 8 ? launch_select<8, false>(a, pl, units, st)
                              : launch_select<16, false>(a, pl, units, st);
  if (rc != MB_OK || pl.cap == 0) return rc;
  for (int64_t u0 = 0; u0 < units; u0 += 65535) {
    // moves only: a part of the units per launch where the grid's second axis ends
    const int64_t nu = std::min<int64_t>(65535, units - u0);
    const int rm = launch_with_pdl(k_evict_move, dim3((pl.cap + kMoveChunk - 1) / kMoveChunk, static_cast<unsigned>(nu)),
                                   dim3(kMoveThreads), 0, st, a, u0);
    if (rm != MB_OK) return rm;
  }
  return MB_OK;
}

}  // extern "C"
