// Eviction from a KV cache by accumulated attention weight on B200 (sm_100a).
//
// Each (layer, trace, KV head) keeps `budget` of its len rows: those whose position is
// recent (>= next_pos - recent) or among the first `sinks`, then the rows of largest
// score, ties to the lowest row. Attention does not depend on the order of a cache's
// rows, so nothing is shifted: the j-th row at or beyond the budget that stays (a mover)
// goes into the j-th row below the budget that leaves (a hole). Holes and movers are
// disjoint, so the moves have no order among them; only moved rows cost bandwidth.
#include <limits.h>

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
__device__ __forceinline__ uint32_t rank_code(float s, int pos, int recent_from, int sinks) {
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
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <int CS>
__device__ __forceinline__ void unit_sync() {
  if (CS > 1)
    cluster_sync();
  else
    __syncthreads();
}

// *word (same place in every CTA) summed over the cluster's lower ranks, and over all of them.
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

constexpr int kBins = 2048;  // most bins of a histogram
constexpr uint32_t kFewRanks = 128;  // compared with one another, one per thread (no CTA is smaller)

// The digit at which the unit's counts, from the largest digit of `bins` downwards, reach `need`;
// how many of that digit are still needed and how many there are. Of a cluster every CTA sums its
// share of the bins over all histograms and leaves the sums with every CTA, in `total` (each CTA
// reading all histograms, 16 units of 8,277 rows took 65 us in place of 26: remote words are the
// bound). The histogram may be written again on return.
template <int CS>
__device__ __forceinline__ void find_digit(const uint32_t* hist, uint32_t* total, int bins, int need, uint32_t* wsum,
                                           int* result) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unit_sync<CS>();
  if (CS > 1) {
    const int share = bins / CS, from = static_cast<int>(cluster_ctarank()) * share;
    for (int i = from + tid; i < from + share; i += blockDim.x) {
      uint32_t x = 0;
#pragma unroll
      for (uint32_t r = 0; r < CS; ++r) x += ld_cluster_u32(mapa_shared(smem_u32(hist + i), r));
#pragma unroll
      for (uint32_t r = 0; r < CS; ++r) st_cluster_u32(mapa_shared(smem_u32(total + i), r), x);
    }
    unit_sync<CS>();
  }
  const uint32_t* sums = CS > 1 ? total : hist;
  const int per = (bins + blockDim.x - 1) / blockDim.x;  // bins of this thread, from the top: at most 16
  const int top = bins - 1 - tid * per;
  uint32_t bin[16];
  int sum = 0;
#pragma unroll
  for (int u = 0; u < 16; ++u) {
    bin[u] = u < per && top - u >= 0 ? sums[top - u] : 0u;
    sum += bin[u];
  }
  int upto = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += x;
  }
  if (lane == 31) wsum[warp] = upto;
  __syncthreads();
  upto += __reduce_add_sync(0xffffffffu, lane < warp ? wsum[lane] : 0u);
  if (upto >= need && upto - sum < need) {  // one thread
    int left = need - (upto - sum), at = 0, count = 0;
    bool done = false;
#pragma unroll
    for (int u = 0; u < 16; ++u)
      if (!done && u < per) {
        at = u;
        count = static_cast<int>(bin[u]);
        done = count >= left;
        if (!done) left -= count;
      }
    result[0] = top - at;
    result[1] = left;
    result[2] = count;
  }
  __syncthreads();
}

// The same for n <= blockDim.x ranks: every thread counts those above its own.
__device__ __forceinline__ void count_above(const uint32_t* cand, int n, int need, int* result) {
  if (static_cast<int>(threadIdx.x) >= n) return;
  const uint32_t mine = cand[threadIdx.x];
  int larger = 0, equal = 0;
  const uint4* c4 = reinterpret_cast<const uint4*>(cand);
#pragma unroll 4
  for (int i = 0; i < n / 4; ++i) {
    const uint4 c = c4[i];
    larger += (c.x > mine) + (c.y > mine) + (c.z > mine) + (c.w > mine);
    equal += (c.x == mine) + (c.y == mine) + (c.z == mine) + (c.w == mine);
  }
  for (int i = n & ~3; i < n; ++i) {
    larger += cand[i] > mine;
    equal += cand[i] == mine;
  }
  if (larger < need && need <= larger + equal) {  // threads of one rank
    result[0] = static_cast<int>(mine);
    result[1] = need - larger;
    result[2] = equal;
  }
}

// And for the last `bits` bits of at most 32 kPer ranks that share the bits above, by one warp:
// the ranks in registers, the answer (the whole rank) bit by bit.
template <int kPer>
__device__ __forceinline__ void finish_in_warp(const uint32_t* cand, int n, uint32_t above, int bits, int need, int lane,
                                               int* result) {
  uint32_t r[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) r[u] = u * 32 + lane < n ? cand[u * 32 + lane] : 0u;  // absent: 0
  uint32_t at = above << bits;
  auto count = [&](auto test) {
    int c = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) c += test(r[u]);
    return __reduce_add_sync(0xffffffffu, c);
  };
  for (int b = bits - 1; b >= 0; --b) {
    const uint32_t trial = at | (1u << b);
    if (count([&](uint32_t x) { return x >= trial; }) >= need) at = trial;
  }
  const int larger = count([&](uint32_t x) { return x > at; });
  const int equal = count([&](uint32_t x) { return x == at; });  // absent ones too if at is 0: more than needed
  if (lane == 0) {
    result[0] = static_cast<int>(at);
    result[1] = need - larger;
    result[2] = equal;
  }
}

// Selection for one (layer, trace, KV head) by a cluster of CS CTAs, each with a slice of the
// rows. Bound by instructions per row where few units share the GPU: scores and positions are
// read once, their ranks stay in shared memory; the kept-th largest rank is found from three
// histograms (joined through distributed shared memory), the second and third of only the rows
// whose first digit is the threshold's (FUSED: those are compared directly where they are few);
// every warp sweeps its own run of rows, so that holes and movers (and ties, where not all of them
// stay) are numbered in row order with one exchange of counts. FUSED (CS = 1): the same CTA moves
// the rows; otherwise the numbered moves go to the workspace for k_evict_move.
// Measured: 4 units of 300 rows 8.3 us, all latency; 6,144 units of 600 to 760 rows of 128, of which 512
// stay, 158 us (90 % of the bytes' time at 6.44 TB/s); 64 units of 60,001 to 65,536 rows, of which 32,768
// stay, 217 us (78 %), 35 of them this kernel.
template <int CS, bool FUSED>
__global__ void __launch_bounds__(FUSED ? 512 : 1024) k_evict(const __grid_constant__ EvictArgs a) {
  extern __shared__ __align__(16) uint32_t dyn[];
  __shared__ uint32_t hist[kBins], total[CS > 1 ? kBins : 1];
  __shared__ uint32_t wsum[kMaxWarps];
  __shared__ int digit[3];
  __shared__ uint32_t n_cand;
  __shared__ uint32_t counts[3][kMaxWarps + 1];  // ties, holes, movers: by warp, then the CTA's
  constexpr int kLow = FUSED ? 22 : 21;  // bits below the first digit
  constexpr int kFirst = 1 << (32 - kLow);
  uint32_t* code = dyn;                  // [slice]
  uint32_t* stay = code + a.slice;       // [slice / 32]
  uint32_t* cand = stay + a.slice / 32;  // [slice / 4] ranks with the threshold's first digit (FUSED)
  const int tid = threadIdx.x, threads = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const uint32_t rank = CS > 1 ? cluster_ctarank() : 0;
  for (int i = tid; i < kFirst; i += threads) hist[i] = 0;
  if (tid == 0) n_cand = 0;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t unit = blockIdx.x / CS;
  const int h = unit % a.Hkv, t = (unit / a.Hkv) % a.T, layer = unit / (static_cast<int64_t>(a.Hkv) * a.T);
  const int len = max(0, min(a.lens[t], a.Lmax));
  const int kept = min(len, a.budget);
  const int recent_from =
      static_cast<int>(max(static_cast<int64_t>(a.next_pos[t]) - a.recent, static_cast<int64_t>(INT_MIN)));
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
      if (4 * i < n) atomicAdd(&hist[c.x >> kLow], 1u);
      if (4 * i + 1 < n) atomicAdd(&hist[c.y >> kLow], 1u);
      if (4 * i + 2 < n) atomicAdd(&hist[c.z >> kLow], 1u);
      if (4 * i + 3 < n) atomicAdd(&hist[c.w >> kLow], 1u);
    }
  } else {
#pragma unroll 4
    for (int i = tid; i < n; i += threads) {
      const uint32_t c = rank_code(sc[r0 + i], ps[r0 + i], recent_from, a.sinks);
      code[i] = c;
      atomicAdd(&hist[c >> kLow], 1u);
    }
  }
  uint32_t first = 0, limit = 0;  // the threshold's first digit; the kept-th largest rank
  int need = kept;
  bool found = FUSED && n <= static_cast<int>(kFewRanks);
  if (found) {
    __syncthreads();
    count_above(code, n, need, digit);
    __syncthreads();
    limit = static_cast<uint32_t>(digit[0]);
  } else {
    find_digit<CS>(hist, total, kFirst, kept, wsum, digit);
    first = digit[0];
    need = digit[1];
  }
  if (FUSED && !found) {  // few rows: those of this digit are usually few enough to be compared
    const uint32_t room = a.slice / 4;
#pragma unroll 4
    for (int i = tid; i < n; i += threads) {
      const uint32_t c = code[i];
      if (c >> kLow == first) {
        const uint32_t at = atomicAdd(&n_cand, 1u);
        if (at < room) cand[at] = c;
      }
    }
    __syncthreads();
    found = n_cand <= min(room, 512u);
    if (found) {
      if (n_cand <= kFewRanks)
        count_above(cand, static_cast<int>(n_cand), need, digit);
      else if (warp == 0)
        finish_in_warp<16>(cand, n_cand, first, kLow, need, lane, digit);
      __syncthreads();
      limit = static_cast<uint32_t>(digit[0]);
    }
  }
  if (!found) {
    auto count_digits = [&](int shift, uint32_t above, int drop, uint32_t mask) {  // of the rows with c >> shift == above
      for (int i = tid; i < kBins; i += threads) hist[i] = 0;
      __syncthreads();
      const uint4* c4 = reinterpret_cast<const uint4*>(code);
#pragma unroll 2
      for (int i = tid; i < (n + 3) / 4; i += threads) {
        const uint4 v = c4[i];
        const uint32_t c[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c[u] >> shift == above && 4 * i + u < n) atomicAdd(&hist[(c[u] >> drop) & mask], 1u);
      }
    };
    count_digits(kLow, first, kLow - 11, kBins - 1);
    find_digit<CS>(hist, total, kBins, need, wsum, digit);
    const uint32_t upper = first << 11 | static_cast<uint32_t>(digit[0]);
    need = digit[1];
    count_digits(kLow - 11, upper, 0, (1u << (kLow - 11)) - 1);
    find_digit<CS>(hist, total, 1 << (kLow - 11), need, wsum, digit);
    limit = upper << (kLow - 11) | static_cast<uint32_t>(digit[0]);
  }
  need = digit[1];
  const bool all_ties = need == digit[2];
  // Every warp's run of rows, whole words of 32; a word's bits are gathered by ballots and then
  // handled by one lane, 32 words at a time.
  const int words = (n + 31) / 32, per = (words + warps - 1) / warps;
  const int w0 = min(words, warp * per), w1 = min(words, w0 + per);
  auto before_lane = [&](int v) {  // sum over the lower lanes
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x - v;
  };
  auto scan = [&](uint32_t* c) {  // counts of the warps before each warp, and of the CTA (one warp)
    const int v = lane < warps ? static_cast<int>(c[lane]) : 0;
    const int x = before_lane(v);
    c[lane] = x;
    if (lane == 31) c[kMaxWarps] = x + v;
  };
  auto gather = [&](int wb, auto test) {  // word wb + lane of this warp's run: bit i is test(row i)
    uint32_t mine = 0;
#pragma unroll 4
    for (int u = 0; u < min(32, w1 - wb); ++u) {
      const int i = (wb + u) * 32 + lane;
      const uint32_t bits = __ballot_sync(0xffffffffu, i < n && test(code[i]));
      mine = u == lane ? bits : mine;
    }
    return mine;
  };
  int all, tie = 0;
  if (!all_ties) {  // the first `need` ties of the unit stay
    int ties = 0;
    for (int wb = w0; wb < w1; wb += 32) ties += __popc(gather(wb, [&](uint32_t c) { return c == limit; }));
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) counts[0][warp] = ties;
    __syncthreads();
    if (warp == 0) scan(counts[0]);
    unit_sync<CS>();
    tie = ranks_before<CS>(&counts[0][kMaxWarps], rank, &all) + counts[0][warp];
  }
  // of word w: the rows below the budget, the valid rows
  auto low_rows = [&](int w) {
    const int below = kept - (r0 + w * 32);
    return below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1;
  };
  auto valid_rows = [&](int w) {
    const int rows = n - w * 32;
    return rows >= 32 ? 0xffffffffu : rows <= 0 ? 0u : (1u << rows) - 1;
  };
  int holes = 0, movers = 0;
  for (int wb = w0; wb < w1; wb += 32) {
    const int w = wb + lane;
    uint32_t bits = gather(wb, [&](uint32_t c) { return c >= limit; });
    if (!all_ties) {
      uint32_t tied = gather(wb, [&](uint32_t c) { return c == limit; });
      const int mine = __popc(tied);
      int spare = need - tie - before_lane(mine);  // ties of this word that stay
      tie += __reduce_add_sync(0xffffffffu, mine);
      for (; tied && spare > 0; --spare) tied &= tied - 1;
      bits &= ~tied;
    }
    if (w < w1) stay[w] = bits;
    const uint32_t low = w < w1 ? low_rows(w) : 0u;
    holes += __popc(valid_rows(w) & low & ~bits);
    movers += __popc(bits & ~low);
  }
  holes = __reduce_add_sync(0xffffffffu, holes);
  movers = __reduce_add_sync(0xffffffffu, movers);
  if (lane == 0) {
    counts[1][warp] = holes;
    counts[2][warp] = movers;
  }
  __syncthreads();
  if (warp < 2) scan(counts[1 + warp]);
  unit_sync<CS>();
  int n_moves;
  const int holes_before = ranks_before<CS>(&counts[1][kMaxWarps], rank, &all);
  const int movers_before = ranks_before<CS>(&counts[2][kMaxWarps], rank, &n_moves);
  // As many rows leave below the budget as stay beyond it. The lists are made in shared memory
  // (FUSED: where they stay; otherwise in the place of the ranks, this CTA's numbers only) and
  // copied out in order: written from here, a lane's few numbers at a time, they took longer than
  // all else but the loads.
  const int cta_holes = static_cast<int>(counts[1][kMaxWarps]), cta_movers = static_cast<int>(counts[2][kMaxWarps]);
  int32_t* hole_list = reinterpret_cast<int32_t*>(FUSED ? cand + a.slice / 4 : code);
  int32_t* mover_list = hole_list + (FUSED ? a.cap : cta_holes);
  int hole = static_cast<int>(counts[1][warp]), mover = static_cast<int>(counts[2][warp]);
  for (int wb = w0; wb < w1; wb += 32) {
    const int w = wb + lane;
    const uint32_t bits = w < w1 ? stay[w] : 0u, low = w < w1 ? low_rows(w) : 0u;
    uint32_t hb = valid_rows(w) & low & ~bits, mb = bits & ~low;
    const int nh = __popc(hb), nm = __popc(mb);
    int at = hole + before_lane(nh);
    for (; hb; hb &= hb - 1) hole_list[at++] = r0 + w * 32 + __ffs(hb) - 1;
    at = mover + before_lane(nm);
    for (; mb; mb &= mb - 1) mover_list[at++] = r0 + w * 32 + __ffs(mb) - 1;
    hole += __reduce_add_sync(0xffffffffu, nh);
    mover += __reduce_add_sync(0xffffffffu, nm);
  }
  if (!FUSED) {
    __syncthreads();
    int32_t* out = a.moves + unit * 2 * a.cap;
    for (int i = tid; i < cta_holes; i += threads) out[holes_before + i] = hole_list[i];
    for (int i = tid; i < cta_movers; i += threads) out[a.cap + movers_before + i] = mover_list[i];
  }
  if (so != sc) {  // what stays below the budget
    const int rows = min(n, kept - r0);
#pragma unroll 4
    for (int i = tid; i < rows; i += threads)
      if ((stay[i >> 5] >> (i & 31)) & 1) {
        so[r0 + i] = sc[r0 + i];
        po[r0 + i] = ps[r0 + i];
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
  // (a second kernel costs more than the moves); its lists lie in shared memory. Measured, one /
  // two kernels: 6,144 units of 760 rows 158 / 246 us, 384 of 4,000 91 / 95, 4 of 300 9.9 / 11.8; but 32 of
  // 2,000 rows, 976 of 128 moved, 16.0 / 12.5.
  pl->fused = Lmax <= 4096 && (units >= 2 * sm_count() || static_cast<int64_t>(pl->cap) * d <= 32 * 1024);
  pl->cs = 1;
  // Enough CTAs per unit to use the SMs, slices that fit; a cluster's exchanges cost more than they
  // save for a few thousand rows. Measured, one CTA / a cluster: 16 units of 8,277 rows 20 / 24 us, 17 of
  // 18,767 32 / 26, 8 of 64,000 49 / 31.
  if (!pl->fused)
    while (pl->cs < 16 && ((Lmax + pl->cs - 1) / pl->cs > kMaxSlice ||
                          (pl->cs < 8 && units * pl->cs * 2 <= sm_count() && Lmax / pl->cs > 8192)))
      pl->cs *= 2;
  pl->slice = ((Lmax + pl->cs - 1) / pl->cs + 127) & ~127;
  if (pl->slice > kMaxSlice) return false;
  pl->threads = pl->slice <= 1024 ? 128 : pl->slice <= 4096 ? 512 : 1024;
  pl->smem = static_cast<size_t>(pl->slice) * 4 + pl->slice / 8 +
             (pl->fused ? pl->slice + static_cast<size_t>(pl->cap) * 8 : 0);
  return true;
}

template <int CS, bool FUSED>
static int launch_select(const EvictArgs& a, const EvictPlan& pl, int64_t units, cudaStream_t st) {
  // whatever the size: of a cluster 17 KB are static
  const int rc = opt_in<k_evict<CS, FUSED>>(200 * 1024, CS > 8);
  if (rc != MB_OK) return rc;
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
  if (cudaLaunchKernelEx(&cfg, k_evict<CS, FUSED>, a) != cudaSuccess) {
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

int32_t mb_cache_evict(const mb_cache_evict_args* g, void* stream) {
  if (!g || !g->k_cache || !g->v_cache || !g->scores || !g->positions || !g->scores_out || !g->positions_out ||
      !g->lens || !g->next_pos || !g->lens_out)
    return MB_ERR_NULL;
  const int layers = g->layers, T = g->T, Hkv = g->Hkv, Lmax = g->Lmax, d = g->d, budget = g->budget;
  if (layers < 1 || T < 1 || Hkv < 1 || Lmax < 1 || d < 1 || budget < 1 || g->recent < 0 || g->sinks < 0)
    return MB_ERR_ARGS;
  if (static_cast<int64_t>(g->recent) + g->sinks > budget) return MB_ERR_ARGS;
  if (g->lens_out == g->lens) return MB_ERR_ARGS;  // every CTA reads the old lengths
  if ((g->scores_out == g->scores) != (g->positions_out == g->positions)) return MB_ERR_ARGS;
  for (const int64_t* s : {g->strides, g->strides + 4})
    if ((layers > 1 && s[0] == 0) || broadcast(s + 1, {T, Hkv, Lmax})) return MB_ERR_ARGS;
  const int64_t units = static_cast<int64_t>(layers) * T * Hkv;
  EvictPlan pl;
  if (units > 0x7FFFFFFll || !evict_plan(units, Lmax, d, budget, &pl)) return MB_ERR_UNSUPPORTED;
  if (!g->workspace || g->workspace_bytes < mb_cache_evict_workspace_size(layers, T, Hkv, Lmax, budget))
    return MB_ERR_WORKSPACE;
  if (!aligned(g->workspace, 16)) return MB_ERR_ALIGN;
  EvictArgs a;
  a.k = g->k_cache;
  a.v = g->v_cache;
  bool vec = d % 8 == 0 && d <= 1024 && aligned(a.k, 16) && aligned(a.v, 16);
  for (int u = 0; u < 4; ++u) {
    a.ks[u] = g->strides[u];
    a.vs[u] = g->strides[4 + u];
  }
  for (int u = 0; u < 8; ++u) vec = vec && g->strides[u] % 8 == 0;
  a.vec = vec;
  a.vec_ranks = Lmax % 4 == 0 && aligned(g->scores, 16) && aligned(g->positions, 16);
  a.scores = g->scores;
  a.positions = g->positions;
  a.scores_out = g->scores_out;
  a.positions_out = g->positions_out;
  a.lens = g->lens;
  a.next_pos = g->next_pos;
  a.lens_out = g->lens_out;
  a.counts = static_cast<int32_t*>(g->workspace);
  a.moves = a.counts + units;
  a.cap = pl.cap;
  a.slice = pl.slice;
  a.layers = layers;
  a.T = T;
  a.Hkv = Hkv;
  a.Lmax = Lmax;
  a.d = d;
  a.budget = budget;
  a.recent = g->recent;
  a.sinks = g->sinks;
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
