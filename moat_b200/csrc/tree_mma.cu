// Tree attention on the fifth-generation tensor cores (sm_100a).
//
// The queries that read one KV head, nodes x heads of its group, form R <= 128 rows (more are cut
// into row blocks); keys come in tiles of 128. Bound by memory where R is small (4 d bytes per key
// for 4 d R operations); the tensor cores and the exponentials (one per row and key, 16 per cycle
// and SM) reach the memory's pace near R = 128. Two kernels share one frame:
//   k_tree_attn_keys (R <= 16) puts the keys on the 128 TMEM lanes,
//     S^T[keys, R] = K Q^T,  O^T[d, R] += V^T P^T,
//   so a tile's exponentials are spread over all threads however few rows there are;
//   k_tree_attn_rows puts the rows there, S[rows, keys] = Q K^T, O[rows, d] += P V, and a thread
//   has one row. V as TMA brings it is the M-major, or N-major, operand: nothing is transposed.
//
// Softmax. A running maximum would have to be exchanged between threads for every tile. Instead a
// row keeps a reference m_ref and p = 2^(x - m_ref) may grow to 2^8 (harmless for the rounding of
// p, whose precision is relative); only when some x exceeds m_ref + 8 (one vote per tile) are the
// maxima taken, m_ref raised and O and the sums rescaled. Sums and O are fp32; p is rounded once, to
// the inputs' type, for its product with V.
//
// Work. The tiles of all (trace, KV head, row block) units, from the device lengths, form one
// sequence that is shared out among one CTA per SM (share_mode): unequal lengths, one long trace and
// many short ones all fill the GPU. A unit inside one CTA is written directly; the pieces of a cut
// unit leave (m_ref, sum, O) in the workspace and k_tree_join adds them in order. No atomics:
// results repeat bit for bit.
//
// Each CTA: softmax warps, a TMA warp that streams K and V tiles through a ring of up to 8 stages, a
// warp that issues score products, one tile ahead of the softmax, and one that issues value
// products. Every wait is bounded; one that gives up sets MB_DEVERR_TIMEOUT and its thread runs
// through without waiting.
//
// Measured on a B200 (calls replayed from a graph; of the 6.44 TB/s of a copy): 16 traces x 16 heads x
// 4,096 rows of 128: R = 1 82.4 us (6.5 TB/s, all of it), R = 16 84.4 us; 8 KV heads, R = 32 45.0, R = 128
// 45.8 us (6.0 TB/s); one trace of 130,001 rows, 8 KV heads, R = 4 87 us (6.1 TB/s); 16 traces of 512 to
// 752 rows, R = 8 22 us (3.9 TB/s: 256 whole units for 148 CTAs, 7 to 18 tiles and starts each where 12.8
// would be even; a CTA with 16 takes about 13 us, starting and ending the rest).
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "tree.cuh"

namespace mb {

constexpr int kTile = 128;  // keys per tile
constexpr int kBox = 32;    // rows per TMA box of a unit's last cached tile: no more boxes than it needs
constexpr int kMaxRows = 128;  // rows of a block
// Up to this many rows the keys fill the TMEM lanes, above it the rows do. Measured, keys / rows: 256
// units of 512 to 752 rows, R = 8 22.2 / 24.0 us; 64 units of 500, R = 8 8.9 / 10.7; R = 16 of 4,096
// rows 84.4 / 83.0, of head dim 64 20.6 / 22.4.
constexpr int kKeysRows = 16;
constexpr int kMaxTraces = 127;  // per launch (the table of their lengths lies in shared memory)
constexpr int kPanel = kTile * 128;  // bytes of a 64-column panel of a tile (128-byte swizzled rows)
constexpr float kNoRef = -1e30f;     // m_ref before any visible key
constexpr float kSlack = 8.0f;       // p may reach 2^kSlack

struct TreeMmaParams {
  TreeAttnArgs a;
  CUtensorMap mq, mk, mv, mk_end, mv_end, mkd, mvd;  // (seven in a row: prefetched by index)
  float* part;  // [2 * grid][rows][DP] unnormalised O of a unit's pieces
  float* ml;    // [2 * grid][2][kMaxRows] their m_ref and sum
  int join_passes;  // rows of a join CTA, in passes of its threads
  bool join_by_unit;
  float* lse;   // [units][kMaxRows] log2 of the softmax denominators (weight pass), or null
  float* kept;  // [units][R][kept_len] scores of the cached rows, kept for the weight pass, or null
  float* kept_draft;  // [units][R][64] of the drafted rows
  int kept_len;
  int t0, T;    // traces of this launch
  int RB, mb, G, grid, nst, nq;
  int n16, used;  // rows of a Q slot; rows of a block in steps of 16
  int tile_cycles, tile_traffic;  // see share_mode
  bool whole;    // every unit in one CTA: nothing to join
  bool vec_out;  // 16-byte pieces of output rows
};

// --- tcgen05 / TMEM -----------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t smem_dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_dst), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// a, b: low words of the operands' descriptors (smem_desc); their high words are alike.
constexpr uint32_t kDescHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void tc_mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
// 16 consecutive TMEM columns of this warp's lanes
__device__ __forceinline__ void tc_ld16(uint32_t addr, float* r) {
  uint32_t u[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void tc_ld4(uint32_t addr, float* r) {
  uint32_t u[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
               : "r"(addr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const float* r) {
  uint32_t u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(r[i]);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}

// Low word of a shared-memory operand with 128-byte swizzle. K-major: rows of 64 elements, 8-row
// groups 1024 bytes apart (lbo unused). MN-major: 64 elements of M or N per 128-byte line, lines
// along K, 8-line groups 1024 bytes apart, the next 64 elements of M or N lbo bytes on.
__device__ __forceinline__ uint32_t smem_desc(uint32_t addr, uint32_t lbo) {
  return ((addr & 0x3FFFF) >> 4) | ((lbo >> 4) << 16);
}
// kind::f16, fp32 accumulator, M = 128; a_mn / b_mn: operand is M- / N-major
__device__ __forceinline__ uint32_t instr_desc(bool bf16, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "l"(policy)
      : "memory");
}

// 16 floats that lie 64-byte aligned in shared memory.
__device__ __forceinline__ void load16(const float* p, float* r) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    r[i] = v.x;
    r[i + 1] = v.y;
    r[i + 2] = v.z;
    r[i + 3] = v.w;
  }
}

// One lane of a converged warp. Branches on it stay uniform for the compiler, so that
// descriptors and addresses live in uniform registers (a test of the lane number made each
// MMA and each TMA instruction cost 100 to 350 cycles to issue).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Largest value over the warp (NaN ignored, as fmaxf does).
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// "Any" over the threads of a named barrier.
__device__ __forceinline__ bool vote_any(bool v, int id, int threads) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(id), "r"(threads)
      : "memory");
  return r != 0;
}

// A wait that can give up: the thread notes it and stops waiting for anything.
__device__ __forceinline__ void guarded_wait(uint64_t* bar, uint32_t parity, bool& dead, uint32_t* err) {
  if (dead) return;
  if (!mbar_wait(bar, parity)) {
    dead = true;
    if (err) atomicOr(err, MB_DEVERR_TIMEOUT);
  }
}

// Sums over the 32 lanes of 16 columns: v[0..16) of every lane in, the sum of column lane % 16
// out.
__device__ __forceinline__ float column_sums16(float* v, int lane) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
#pragma unroll
  for (int o = 8; o; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = up ? v[i] : v[i + o];
      const float keep = up ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

// --- the sequence of tiles ------------------------------------------------------
// Tiles of trace t per unit: its committed rows, then one tile of drafted rows.
__device__ __forceinline__ int trace_len(const TreeAttnArgs& a, int t) { return max(0, min(a.lens[t], a.Lmax)); }
__device__ __forceinline__ int trace_tiles(int len) { return (len + kTile - 1) / kTile + 1; }

// First position of CTA c of g when a sequence of w is cut evenly.
// (floor(w c / g), without its 64-bit division: that took a CTA's set-up 0.2 us.)
__device__ __forceinline__ int cut(uint32_t w, uint32_t c, uint32_t g) {
  const uint32_t q = w / g;
  return static_cast<int>(q * c + (w - q * g) * c / g);
}

struct Segment {  // a run of tiles of one unit
  int t, kvh, rb, len, nt, j0, n;
};

// Lengths of the launch's traces and where each begins in the sequence, in shared memory.
struct TraceTable {
  int cum[kMaxTraces + 1];
  int len[kMaxTraces];
  int max_span;
};

// Starting and ending a piece costs about as much as a tile; it counts as one in the sequence,
// before the unit's first tile (without it a CTA with many short units finished last by 3x).
constexpr int kUnitCost = 1;

__device__ __forceinline__ int unit_span(int nt) { return nt + kUnitCost; }

// The next segment at or after position f of the sequence (RB row blocks per trace and KV head);
// moves f past it. False at the end of this CTA's share.
__device__ __forceinline__ bool next_segment(const TreeMmaParams& p, const TraceTable& tab, int& f, int end, int RB,
                                             Segment& s) {
  while (f < end) {
    int lo = 0, hi = p.T - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tab.cum[mid] <= f)
        lo = mid;
      else
        hi = mid - 1;
    }
    s.t = p.t0 + lo;
    s.len = tab.len[lo];
    s.nt = trace_tiles(s.len);
    const int span = unit_span(s.nt), rem = f - tab.cum[lo], u = rem / span;
    const int tile0 = tab.cum[lo] + u * span + kUnitCost;  // position of the unit's first tile
    s.kvh = u / RB;
    s.rb = u - s.kvh * RB;
    s.j0 = max(0, f - tile0);
    s.n = min(s.nt, end - tile0) - s.j0;
    f = s.n > 0 ? tile0 + s.j0 + s.n : end;
    if (s.n > 0) return true;
  }
  return false;
}

// Valid rows of tile j of a unit (its last tile holds the drafted rows).
__device__ __forceinline__ int tile_rows(int len, int nt, int m, int j) {
  return j == nt - 1 ? m : min(kTile, len - j * kTile);
}

// Fills the table (warp 0) for `units` units per trace.
__device__ __forceinline__ void prefix_tiles(const TreeMmaParams& p, TraceTable& tab, int lane, int units) {
  int base = 0, longest = 0;
  for (int c = 0; c < p.T; c += 32) {
    const int t = c + lane;
    const int len = t < p.T ? trace_len(p.a, p.t0 + t) : 0;
    longest = max(longest, len);
    int v = t < p.T ? unit_span(trace_tiles(len)) * units : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (t < p.T) {
      tab.cum[t + 1] = base + v;
      tab.len[t] = len;
    }
    base += __shfl_sync(0xffffffffu, v, 31);
  }
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 0) {
    tab.cum[0] = 0;
    tab.max_span = unit_span(trace_tiles(longest));
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool BF16>
__device__ __forceinline__ uint16_t round16(float x) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}

// Shared memory: ring | Q slots | P (rows kernel: outputs on their way) | barriers and small tables.
struct TreeSmem {
  uint32_t ring, q, p, stage, qslot;  // byte offsets, bytes per stage / slot
  uint32_t misc, total;
};
constexpr int kMaxStages = 8;
constexpr uint32_t kMiscBars = 256;                          // barriers, TMEM base, noted rows
constexpr uint32_t kMiscNoted = 240;
constexpr uint32_t kMiscRef = kMiscBars;                     // m_ref [128]
constexpr uint32_t kMiscMask = kMiscRef + kMaxRows * 4;      // draft masks by row [128]
constexpr uint32_t kMiscTab = kMiscMask + kMaxRows * 8;      // TraceTable
constexpr uint32_t kMiscBytes = kMiscTab + sizeof(TraceTable);

__host__ __device__ inline TreeSmem tree_smem(int panels, int n16, int nst, int nq) {
  TreeSmem s;
  s.stage = panels * kPanel;
  s.qslot = panels * n16 * 128;
  s.ring = 0;
  s.q = s.ring + nst * s.stage;
  s.p = s.q + nq * s.qslot;
  s.misc = s.p + kPanel;
  s.total = s.misc + kMiscBytes;
  return s;
}

// Rows R .. n16 - 1 of every panel of the Q slots: the boxes never write them, they stay zero.
__device__ __forceinline__ void zero_query_tail(uint8_t* q, int panels, int n16, int R, int tid, int threads) {
  const int per = (n16 - R) * 8;  // 16-byte pieces per panel
  for (int i = tid; i < panels * per; i += threads) {
    const int pn = i / per;
    *reinterpret_cast<uint4*>(q + (pn * n16 + R) * 128 + (i - pn * per) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}

// How the sequence is shared out. Cutting units evenly costs their pieces' way through the workspace
// and the join, 2 to 12 us; whole units cost idle CTAs at the end, which does not matter while the
// memory is the bound. A tile takes a CTA p.tile_cycles; the memory needs p.tile_traffic cycles for
// the tiles of one position in every CTA. Whole units are kept as long as the longest share of them,
// with kShareFixed cycles for starting and ending, ends before the traffic does. Measured, 16 traces
// of 4,096 rows of 128: 128 units of 128 / 32 rows 47.5 / 45.7 us whole, 55.7 / 47.6 cut; 256 units of 8
// rows 84.4 dealt out whole, 88.2 cut; 256 units of 512 to 752 rows 22.7 and 22.4; of a few long units
// only pieces fill the GPU.
// Units so short that the longest share of whole ones outlasts the even one by less than a join
// takes, kJoinCycles, are not cut either. Measured, whole / cut: 128 units of 200 to 300 rows 9.7 / 13.6 us,
// 256 of them 15.7 / 19.0, 100 units of 300 to 620 rows and 64 query rows 12.9 / 17.8, 32 units of 500 to 700
// rows 10.3 / 11.2.
enum class Share { kCut, kWholeUnit, kSnapped };
constexpr int kShareFixed = 12000, kJoinCycles = 12000;

__device__ __forceinline__ Share share_mode(const TreeMmaParams& p, int64_t total, int64_t max_span, int units) {
  if (p.whole) return Share::kWholeUnit;
  const int64_t traffic = p.tile_traffic * total - static_cast<int64_t>(kShareFixed) * p.grid;  // x grid CTAs
  const int64_t longest = max_span * p.tile_cycles * p.grid;
  if (units <= p.grid)
    return longest <= traffic || (max_span - total / p.grid) * p.tile_cycles <= kJoinCycles ? Share::kWholeUnit
                                                                                            : Share::kCut;
  return longest + p.tile_cycles * total <= traffic || max_span * p.tile_cycles <= kJoinCycles ? Share::kSnapped
                                                                                                 : Share::kCut;
}

// The unit boundary nearest to position f.
__device__ __forceinline__ int snap(const TreeMmaParams& p, const TraceTable& tab, int f) {
  int lo = 0, hi = p.T;  // cum[T] is a boundary too
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.cum[mid] <= f)
      lo = mid;
    else
      hi = mid - 1;
  }
  if (lo == p.T) return f;
  const int span = unit_span(trace_tiles(tab.len[lo]));
  return tab.cum[lo] + (f - tab.cum[lo] + span / 2) / span * span;
}

// Positions of the sequence that are CTA c's.
__device__ __forceinline__ void cta_share(const TreeMmaParams& p, const TraceTable& tab, int c, int* beg, int* end) {
  *beg = *end = 0;
  const int units = p.a.Hkv * p.RB, total = tab.cum[p.T], g = min(p.grid, total);
  const Share mode = share_mode(p, total, tab.max_span, units * p.T);
  if (mode == Share::kWholeUnit) {
    const int t = c / units;
    if (t >= p.T) return;
    const int span = unit_span(trace_tiles(tab.len[t]));
    *beg = tab.cum[t] + (c - t * units) * span;
    *end = *beg + span;
  } else if (c < g) {  // CTAs with work
    *beg = cut(total, c, g);
    *end = cut(total, c + 1, g);
    if (mode == Share::kSnapped) {
      *beg = snap(p, tab, *beg);
      *end = snap(p, tab, *end);
    }
  }
}

struct TreeBars {
  uint64_t *kv_full, *kv_empty, *q_full, *q_empty;
};

// The TMA warp: K and V tiles of this CTA's segments through the ring, a segment's queries
// before them, or after its first tile when their slot may still be in use.
template <int PANELS>
__device__ __forceinline__ void tma_role(const TreeMmaParams& p, const TraceTable& tab, const TreeSmem& lay,
                                         const TreeBars& bars, int beg, int end, uint32_t ring, uint32_t qbase, int R) {
  const TreeAttnArgs& a = p.a;
  bool dead = false;
  // a cache that is read once streams past what L2 should keep; several row blocks or the
  // weight pass read it again
  uint64_t policy;
  if (p.RB == 1 && (!p.lse || p.kept))
    policy = policy_evict_first();
  else
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(policy));
  const uint64_t keep = policy_evict_last();
  int item = 0, seg = 0, st = 0, use = 0;  // K and V tiles of the ring (stage, times used), segments
  Segment s;
  for (int f = beg; next_segment(p, tab, f, end, p.RB, s); ++seg) {
    const int qs = p.nq == 2 ? seg & 1 : 0, quse = p.nq == 2 ? seg >> 1 : seg;
    auto load_queries = [&] {
      if (elect_one()) {
        mbar_expect_tx(bars.q_full + qs, PANELS * R * 128);
        for (int pn = 0; pn < PANELS; ++pn)
          tma_load_4d(qbase + qs * lay.qslot + pn * p.n16 * 128, &p.mq, bars.q_full + qs, pn * 64, s.kvh * p.G,
                      s.rb * p.mb, s.t, keep);
      }
      __syncwarp();
    };
    if (quse == 0) load_queries();
    for (int j = s.j0; j < s.j0 + s.n; ++j) {
      const bool draft = j == s.nt - 1;
      const int rows = tile_rows(s.len, s.nt, a.m, j);
      for (int kv = 0; kv < 2; ++kv, ++item) {
        if (use > 0) guarded_wait(bars.kv_empty + st, (use - 1) & 1, dead, a.err);
        const uint32_t dst = ring + st * lay.stage;
        if (elect_one()) {
          if (draft) {
            mbar_expect_tx(bars.kv_full + st, PANELS * 128 * a.m);
            for (int pn = 0; pn < PANELS; ++pn)
              tma_load_4d(dst + pn * kPanel, kv ? &p.mvd : &p.mkd, bars.kv_full + st, pn * 64, s.kvh, 0, s.t, keep);
          } else if (rows == kTile) {
            mbar_expect_tx(bars.kv_full + st, PANELS * kPanel);
            for (int pn = 0; pn < PANELS; ++pn)
              tma_load_4d(dst + pn * kPanel, kv ? &p.mv : &p.mk, bars.kv_full + st, pn * 64, j * kTile, s.kvh, s.t,
                          policy);
          } else {
            const int boxes = (rows + kBox - 1) / kBox;
            mbar_expect_tx(bars.kv_full + st, PANELS * 128 * boxes * kBox);
            for (int pn = 0; pn < PANELS; ++pn)
              for (int b = 0; b < boxes; ++b)
                tma_load_4d(dst + pn * kPanel + b * kBox * 128, kv ? &p.mv_end : &p.mk_end, bars.kv_full + st, pn * 64,
                            j * kTile + b * kBox, s.kvh, s.t, policy);
          }
        }
        __syncwarp();
        if (++st == p.nst) {
          st = 0;
          ++use;
        }
      }
      if (quse > 0 && j == s.j0) {
        guarded_wait(bars.q_empty + qs, (quse - 1) & 1, dead, a.err);
        load_queries();
      }
    }
  }
  if (dead)  // copies still in flight must land before this CTA's shared memory goes
    for (int i = max(0, item - p.nst); i < item; ++i) mbar_wait(bars.kv_full + i % p.nst, (i / p.nst) & 1);
}

// The next tile's stage: every other item of the ring.
__device__ __forceinline__ void next_tile(int nst, int& st, int& use) {
  st += 2;
  if (st >= nst) {
    st -= nst;
    ++use;
  }
}

// After a wait gave up: products still in flight must end before TMEM is freed.
__device__ __forceinline__ void drain_products() {
  const long long t0 = clock64();
  while (clock64() - t0 < 1000000) {
  }
}

// Masks of a trace for a segment, two per lane of a warp (node lane and lane + 32). Loads are
// volatile: the compiler moved them down to the drafted tile that uses them, which then took 2,700
// cycles instead of 300.
struct SegmentMasks {
  uint64_t lo, hi;
};

__device__ __forceinline__ uint64_t ld_mask(const uint64_t* p) {
  uint64_t v;
  asm volatile("ld.global.u64 %0, [%1];" : "=l"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ SegmentMasks load_masks(const TreeAttnArgs& a, int t, int lane) {
  const uint64_t* mk = a.masks + t * a.mask_stride;
  SegmentMasks m;
  m.lo = lane < a.m ? ld_mask(mk + lane) : 0;
  m.hi = lane + 32 < a.m ? ld_mask(mk + lane + 32) : 0;
  return m;
}

// Drafted rows that any node sees, one bit each (a warp's masks together are the trace's).
__device__ __forceinline__ uint64_t rows_in_use(const SegmentMasks& m) {
  const uint64_t u = m.lo | m.hi;
  const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(u));
  const uint32_t hi = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(u >> 32));
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// A value that is not finite must not reach a node that does not see its row, but in the product
// with V it would (0 x inf is NaN). So the drafted rows, the only ones that some nodes see and
// others do not, are looked through: what is not finite becomes 0 in shared memory, the row is
// noted, and the output's end adds it for the nodes that see it.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {  // bits 15 and 31: the low, the high half
  constexpr uint32_t e = BF16 ? 0x7F807F80u : 0x7C007C00u, one = BF16 ? 0x00800080u : 0x04000400u;
  return ((x & e) + one) & 0x80008000u;
}
template <bool BF16>
__device__ __forceinline__ bool not_finite(uint16_t x) {
  return (not_finite2<BF16>(x) & 0x8000u) != 0;
}

// Makes a V tile fit for its product, by the warp that issues it (idle until P is there; done by
// the softmax warps it cost them 300 to 1,000 cycles per unit): lines beyond the valid rows in the
// last 16-row step, and drafted rows that no node sees, may hold anything and become 0; of the other
// drafted rows what is not finite does, and noted[0..1] gets their bits.
template <int PANELS, bool BF16>
__device__ __forceinline__ void prepare_values(uint8_t* tile, int rows, bool draft, const SegmentMasks& masks, int lane,
                                               volatile uint32_t* noted) {
  auto piece = [&](int line, int i) {  // 16 bytes: piece i of a line's PANELS * 8
    return reinterpret_cast<uint4*>(tile + (i >> 3) * kPanel + line * 128 + (i & 7) * 16);
  };
  const int end = (rows + 15) & ~15;
  for (int i = lane; i < (end - rows) * PANELS * 8; i += 32)
    *piece(rows + i / (PANELS * 8), i % (PANELS * 8)) = make_uint4(0, 0, 0, 0);
  if (draft) {
    uint64_t unused = ~rows_in_use(masks) & (rows == 64 ? ~0ull : (1ull << rows) - 1);
    for (; unused; unused &= unused - 1)
      if (lane < PANELS * 8) *piece(__ffsll(unused) - 1, lane) = make_uint4(0, 0, 0, 0);
    __syncwarp();
    uint32_t bad = 0;
#pragma unroll 4
    for (int i = lane; i < rows * PANELS * 8; i += 32) {
      const uint4 x = *piece(i / (PANELS * 8), i % (PANELS * 8));
      bad |= not_finite2<BF16>(x.x) | not_finite2<BF16>(x.y) | not_finite2<BF16>(x.z) | not_finite2<BF16>(x.w);
    }
    uint32_t lo = 0, hi = 0;
    if (__any_sync(0xffffffffu, bad != 0)) {  // rare: line by line
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        bool found = false;
        if (lane < PANELS * 8) {
          uint4 x = *piece(r, lane);
          uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t b = not_finite2<BF16>(w[u]);
            found |= b != 0;
            w[u] &= ~((b >> 15) * 0xFFFFu);
          }
          *piece(r, lane) = x;
        }
        const uint32_t bit = __any_sync(0xffffffffu, found) ? 1u << (r & 31) : 0u;
        if (r < 32)
          lo |= bit;
        else
          hi |= bit;
      }
    }
    if (lane == 0) {
      noted[0] = lo;
      noted[1] = hi;
    }
    __threadfence_block();
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// The sum over the noted rows in `rows` that are not finite at head-dim position c of trace t's
// drafted values (0 if all are).
template <bool BF16>
__device__ __noinline__ float noted_values(const TreeAttnArgs& a, int t, int kvh, uint64_t rows, int c) {
  float sum = 0.0f;
  for (; rows; rows &= rows - 1) {
    const uint16_t v = a.vd[t * a.vds[0] + (__ffsll(rows) - 1) * a.vds[1] + kvh * a.vds[2] + c];
    if (not_finite<BF16>(v))
      sum += BF16 ? __uint_as_float(static_cast<uint32_t>(v) << 16) : __half2float(__ushort_as_half(v));
  }
  return sum;
}

// Adds them to columns c0 .. c1 - 1 of an output row, of either form.
template <bool BF16>
__device__ __noinline__ void add_noted(const TreeAttnArgs& a, int t, int kvh, uint64_t rows, uint16_t* out, float* part,
                                       int c0, int c1) {
  for (int c = c0; c < c1; ++c) {
    const float v = noted_values<BF16>(a, t, kvh, rows, c);
    if (v == 0.0f) continue;
    if (part)
      part[c] += v;
    else
      out[c] = round16<BF16>((BF16 ? __uint_as_float(static_cast<uint32_t>(out[c]) << 16)
                                   : __half2float(__ushort_as_half(out[c]))) + v);
  }
}

// ---------------------------------------------------------------------------
// Up to 16 rows: the keys fill the TMEM lanes.
// PANELS: 64-column panels of the head dim (1: d <= 64, 2: d <= 128).
// ---------------------------------------------------------------------------
constexpr int kKeysThreads = 128 + 96;  // softmax, TMA, score products, value products

template <int PANELS, bool BF16>
__global__ void __launch_bounds__(kKeysThreads, 1) k_tree_attn_keys(const __grid_constant__ TreeMmaParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int DP = PANELS * 64;
  constexpr int kSoft = 128;
  const TreeSmem lay = tree_smem(PANELS, p.n16, p.nst, p.nq);
  uint8_t* misc = smem + lay.misc;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(misc);  // [kMaxStages]
  uint64_t* kv_empty = kv_full + kMaxStages;              // [kMaxStages]
  uint64_t* s_full = kv_empty + kMaxStages;               // [2]
  uint64_t* s_empty = s_full + 2;                         // [2]
  uint64_t* q_full = s_empty + 2;                         // [2]
  uint64_t* q_empty = q_full + 2;                         // [2]
  uint64_t* o_empty = q_empty + 2;                        // [2]
  const TreeBars bars = {kv_full, kv_empty, q_full, q_empty};
  uint64_t* p_full = o_empty + 2;
  uint64_t* pv_done = p_full + 1;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(pv_done + 1);
  float* ref = reinterpret_cast<float*>(misc + kMiscRef);
  uint64_t* rowmask = reinterpret_cast<uint64_t*>(misc + kMiscMask);
  TraceTable& tab = *reinterpret_cast<TraceTable*>(misc + kMiscTab);
  // drafted rows, see prepare_values: two segments' (the next one's value warp may be ahead)
  volatile uint32_t* noted = reinterpret_cast<uint32_t*>(misc + kMiscNoted);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TreeAttnArgs& a = p.a;
  const int R = p.mb * p.G;
  bool dead = false;

  if (warp == 4) {  // TMA warp
    if (lane < 7) prefetch_map(&p.mq + lane);
    if (lane == 0) {
      for (int i = 0; i < kMaxStages; ++i) {
        mbar_init(kv_full + i, 1);
        mbar_init(kv_empty + i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + i, 1);
        mbar_init(s_empty + i, kSoft);
        mbar_init(q_full + i, 1);
        mbar_init(q_empty + i, 1);
        mbar_init(o_empty + i, kSoft);
      }
      mbar_init(p_full, kSoft);
      mbar_init(pv_done, 1);
      fence_mbar_init();
    }
  } else if (warp == 5) {
    tmem_alloc(smem_u32(tmem_base), 128);
  } else if (warp < 4) {
    zero_query_tail(smem + lay.q, PANELS * p.nq, p.n16, R, tid, kSoft);
    if (tid < kKeysRows) ref[tid] = kNoRef;
  }
  pdl_wait();  // the lengths, masks, queries and drafts may come from the kernel before
  pdl_launch_dependents();
  tc_before_sync();
  if (warp == 4) {  // builds the table and goes straight on to its loads
    prefix_tiles(p, tab, lane, a.Hkv * p.RB);
    __syncwarp();
    asm volatile("bar.arrive 2, %0;" ::"n"(kKeysThreads) : "memory");
  } else {
    named_bar_sync(2, kKeysThreads);
  }
  tc_after_sync();
  const int c = blockIdx.x;
  int beg, end;
  cta_share(p, tab, c, &beg, &end);
  const uint32_t ring = smem_u32(smem + lay.ring), qbase = smem_u32(smem + lay.q), pbase = smem_u32(smem + lay.p);

  if (warp == 4) {
    tma_role<PANELS>(p, tab, lay, bars, beg, end, ring, qbase, R);
  } else if (warp == 5) {
    // ---------------------------------------------------------------- scores
    const uint32_t idesc = instr_desc(BF16, kKeysRows, false, false);
    const uint32_t ring_k = smem_desc(ring, 16), q_desc = smem_desc(qbase, 16);
    const uint32_t tmem = *tmem_base;
    int k = 0, seg = 0, st = 0, use = 0;  // tile k's K and V are items 2k and 2k + 1 of the ring
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, p.RB, s); ++seg) {
      const int qs = seg & 1;
      guarded_wait(q_full + qs, (seg >> 1) & 1, dead, a.err);
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        guarded_wait(kv_full + st, use & 1, dead, a.err);
        if (k >= 2) guarded_wait(s_empty + (k & 1), ((k >> 1) - 1) & 1, dead, a.err);
        tc_after_sync();
        if (elect_one()) {
          const uint32_t ka = ring_k + (st * lay.stage >> 4), qb = q_desc + (qs * lay.qslot >> 4);
#pragma unroll
          for (int kk = 0; kk < PANELS * 4; ++kk)
            tc_mma(tmem + (k & 1) * kKeysRows, ka + (kk >> 2) * (kPanel >> 4) + (kk & 3) * 2,
                   qb + (kk >> 2) * (kKeysRows * 128 >> 4) + (kk & 3) * 2, idesc, kk > 0);
          tc_commit(s_full + (k & 1));
          tc_commit(kv_empty + st);
          if (jj + 1 == s.n) tc_commit(q_empty + qs);
        }
        __syncwarp();
        next_tile(p.nst, st, use);
      }
    }
    if (dead) drain_products();
  } else if (warp == 6) {
    // ---------------------------------------------------------------- values
    // (a warp of its own: one that issued both products was busy 1,500 cycles a tile, and a
    // score product that had to wait for its keys held back a value product that had not)
    const uint32_t idesc = instr_desc(BF16, kKeysRows, true, true);
    const uint32_t ring_v = smem_desc(ring, kPanel), p_desc = smem_desc(pbase, kPanel);
    const uint32_t tmem = *tmem_base;
    int k = 0, seg = 0, st = 1, use = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, p.RB, s); ++seg) {
      const uint32_t o = tmem + (2 + (seg & 1)) * kKeysRows;
      const SegmentMasks masks = load_masks(a, s.t, lane);
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        const bool draft = s.j0 + jj == s.nt - 1;
        const int rows = tile_rows(s.len, s.nt, a.m, s.j0 + jj), steps = (rows + 15) / 16;
        guarded_wait(kv_full + st, use & 1, dead, a.err);
        if (rows & 15 || draft)
          prepare_values<PANELS, BF16>(smem + lay.ring + st * lay.stage, rows, draft, masks, lane, noted + 2 * (seg & 1));
        if (jj == 0 && seg >= 2) guarded_wait(o_empty + (seg & 1), ((seg >> 1) - 1) & 1, dead, a.err);
        guarded_wait(p_full, k & 1, dead, a.err);
        tc_after_sync();
        if (elect_one()) {
          const uint32_t va = ring_v + (st * lay.stage >> 4);
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            if (kk < steps) tc_mma(o, va + kk * (2048 >> 4), p_desc + kk * (2048 >> 4), idesc, jj > 0 || kk > 0);
          tc_commit(kv_empty + st);
          tc_commit(pv_done);
        }
        __syncwarp();
        next_tile(p.nst, st, use);
      }
    }
    if (dead) drain_products();
  } else {
    // ---------------------------------------------------------------- softmax
    const int wq = warp;
    const int key = wq * 32 + lane;  // this thread's key of a tile, and its d of O^T
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const float sc = a.scale_log2;
    const int my_node = tid / p.G;  // node of row tid
    float l[kKeysRows];
#pragma unroll
    for (int i = 0; i < kKeysRows; ++i) l[i] = 0.0f;
    float* scratch = reinterpret_cast<float*>(smem + lay.p);  // P's space, while no product reads it
    const uint32_t tmem = *tmem_base;
    int seg = 0, k = 0;
    Segment s, next;
    uint64_t mask = 0, next_mask = 0;  // of row tid
    int f = beg;
    bool more = next_segment(p, tab, f, end, p.RB, s);
    auto mask_of = [&](const Segment& g) {  // few rows are one block
      return tid < R ? ld_mask(a.masks + g.t * a.mask_stride + my_node) : 0;
    };
    if (more) mask = mask_of(s);
    for (; more; ++seg, s = next, mask = next_mask) {
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        const int j = s.j0 + jj;
        const bool draft = j == s.nt - 1;
        const int rows = tile_rows(s.len, s.nt, a.m, j);
        const uint32_t sbuf = tmem + lanes + (k & 1) * kKeysRows;
        // which of this thread's rows see its key, a bit each
        uint32_t see = key < rows ? ~0u : 0u;
        if (draft) {
          if (tid < kKeysRows) rowmask[tid] = mask;
          named_bar_sync(1, kSoft);
          if (key < rows) {
            see = 0;
#pragma unroll 4
            for (int i = 0; i < kKeysRows; ++i) see |= static_cast<uint32_t>((rowmask[i] >> key) & 1) << i;
          }
        }
        const bool full = !draft && rows == kTile;
        // the rows' scores of this key, less m_ref (log2 units), -inf for what a row does not see
        float x[kKeysRows], r[kKeysRows];
        auto form = [&](bool less_ref) {
          if (less_ref) load16(ref, r);
          tc_ld16(sbuf, x);
          tc_wait_ld();
#pragma unroll
          for (int u = 0; u < kKeysRows; ++u) x[u] = less_ref ? fmaf(x[u], sc, -r[u]) : x[u] * sc;
          if (!full) {
#pragma unroll
            for (int u = 0; u < kKeysRows; ++u) x[u] = (see >> u) & 1 ? x[u] : -INFINITY;
          }
        };
        guarded_wait(s_full + (k & 1), (k >> 1) & 1, dead, a.err);
        tc_after_sync();
        bool raise = jj == 0;  // a piece's first tile always sets m_ref
        if (!raise) {
          form(true);
          float top = x[0];
#pragma unroll
          for (int u = 1; u < kKeysRows; ++u) top = fmaxf(top, x[u]);
          raise = vote_any(top > kSlack, 1, kSoft);
        }
        if (raise) {
          // P's space and O are free once the previous value product has finished
          if (k > 0) guarded_wait(pv_done, (k - 1) & 1, dead, a.err);
          tc_after_sync();
          form(false);
          float mine = 0.0f;
#pragma unroll
          for (int u = 0; u < kKeysRows; ++u) {
            const float mx = warp_max(x[u]);
            if (u == lane) mine = mx;
          }
          if (lane < kKeysRows) scratch[wq * kKeysRows + lane] = mine;
          named_bar_sync(1, kSoft);
          if (tid < kKeysRows) {
            const float old = ref[tid];
            float mx = old;
#pragma unroll
            for (int w = 0; w < 4; ++w) mx = fmaxf(mx, scratch[w * kKeysRows + tid]);
            ref[tid] = mx;
            scratch[4 * kKeysRows + tid] = ex2(old - mx);
          }
          named_bar_sync(1, kSoft);
          if (jj > 0) {
            const uint32_t ob = tmem + lanes + (2 + (seg & 1)) * kKeysRows;
            load16(scratch + 4 * kKeysRows, r);
#pragma unroll
            for (int u = 0; u < kKeysRows; ++u) l[u] *= r[u];
            tc_ld16(ob, x);
            tc_wait_ld();
#pragma unroll
            for (int u = 0; u < kKeysRows; ++u) x[u] *= r[u];
            tc_st16(ob, x);
            tc_wait_st();
          }
          named_bar_sync(1, kSoft);  // scratch read: its space becomes P again
          form(true);
        }
        tc_before_sync();
        mbar_arrive(s_empty + (k & 1));
        if (p.kept && key < rows) {  // the score itself, for the weight pass
          const int64_t unit = static_cast<int64_t>(s.t) * a.Hkv + s.kvh;
          const int64_t step = draft ? 64 : p.kept_len;
          float* keep = draft ? p.kept_draft + unit * R * 64 + key : p.kept + unit * R * p.kept_len + j * kTile + key;
#pragma unroll
          for (int u = 0; u < kKeysRows; ++u)
            if (u < R) keep[u * step] = x[u] + r[u];
        }
        // p = 2^(x - m_ref), one rounding to the inputs' type for the product with V
        uint32_t pk[kKeysRows / 2];
#pragma unroll
        for (int u = 0; u < kKeysRows; u += 2) {
          const float e0 = ex2(x[u]), e1 = ex2(x[u + 1]);
          l[u] += e0;
          l[u + 1] += e1;
          pk[u / 2] = pack2<BF16>(e0, e1);
        }
        if (k > 0) guarded_wait(pv_done, (k - 1) & 1, dead, a.err);  // P's space is free
        uint8_t* prow = smem + lay.p + key * 128;
        *reinterpret_cast<uint4*>(prow + ((key & 7) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        *reinterpret_cast<uint4*>(prow + ((1 ^ (key & 7)) << 4)) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
        fence_proxy_async_smem();
        tc_before_sync();
        mbar_arrive(p_full);
      }
      // ------------------------------------------------ end of the segment: sums, output
      more = next_segment(p, tab, f, end, p.RB, next);  // under the last value product
      if (more) next_mask = mask_of(next);
      const float part_sum = column_sums16(l, lane);
      guarded_wait(pv_done, (k - 1) & 1, dead, a.err);
      tc_after_sync();
      if (lane < kKeysRows) scratch[wq * kKeysRows + lane] = part_sum;
      named_bar_sync(1, kSoft);
      const bool whole = s.n == s.nt;
      const int slot = 2 * c + (s.j0 > 0 ? 0 : 1);
      if (tid < kKeysRows) {
        const float sum = (scratch[tid] + scratch[kKeysRows + tid]) + (scratch[2 * kKeysRows + tid] +
                                                                       scratch[3 * kKeysRows + tid]);
        const bool real = mask != 0 && sum != 0.0f;
        const float top = ref[tid];
        scratch[4 * kKeysRows + tid] = real ? 1.0f / sum : 0.0f;  // 0 marks a row without keys
        ref[tid] = kNoRef;
        if (!whole) {
          float* ml = p.ml + static_cast<int64_t>(slot) * 2 * kMaxRows;
          ml[tid] = top;
          ml[kMaxRows + tid] = real ? sum : 0.0f;
        } else if (p.lse) {
          const int64_t unit = static_cast<int64_t>(s.t) * a.Hkv + s.kvh;
          p.lse[unit * kMaxRows + tid] = real ? top + log2f(sum) : INFINITY;
        }
      }
      named_bar_sync(1, kSoft);
      const uint32_t ob = tmem + lanes + (2 + (seg & 1)) * kKeysRows;
      const volatile uint32_t* nt = noted + 2 * (seg & 1);
      const uint64_t bad = s.j0 + s.n == s.nt ? static_cast<uint64_t>(nt[1]) << 32 | nt[0] : 0;
      int row = 0, nd = 0, gh = 0;  // row, its node, its head of the group
      uint16_t* out = a.out + s.t * a.os[0] + s.kvh * p.G * a.os[2] + key;
      float* part = p.part + static_cast<int64_t>(slot) * R * DP + key;
#pragma unroll 1
      for (int i = 0; i < R; i += 4) {
        float o[4];
        tc_ld4(ob + i, o);
        const float4 inv = *reinterpret_cast<const float4*>(scratch + 4 * kKeysRows + row);
        tc_wait_ld();
#pragma unroll
        for (int u = 0; u < 4; ++u, ++row) {
          const float scale = u == 0 ? inv.x : u == 1 ? inv.y : u == 2 ? inv.z : inv.w;
          if (row < R) {
            if (bad && (bad & rowmask[row]) && key < a.d)
              o[u] += noted_values<BF16>(a, s.t, s.kvh, bad & rowmask[row], key);
            if (!whole) {
              if (key < DP) *part = o[u];
              part += DP;
            } else {
              if (key < a.d) *out = round16<BF16>(scale == 0.0f ? 0.0f : o[u] * scale);
              out += a.os[2];
              if (++gh == p.G) {
                gh = 0;
                ++nd;
                out += a.os[1] - p.G * a.os[2];
              }
            }
          }
        }
      }
      tc_before_sync();
      mbar_arrive(o_empty + (seg & 1));
#pragma unroll
      for (int i = 0; i < kKeysRows; ++i) l[i] = 0.0f;
      named_bar_sync(1, kSoft);  // scratch read, m_ref reset
    }
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (warp == 5) tmem_dealloc(*tmem_base, 128);
}

// ---------------------------------------------------------------------------
// More than 16 rows: the rows fill the TMEM lanes (S[128 rows, 128 keys], O[128 rows, d]).
// A thread holds 64 scores of one row, so the running reference, the sum and the mask are one
// register each. Either half of a tile's keys belongs to four warps of its own with their own
// reference, sums and O (added with their factors when the segment ends), so that no warp waits
// for another within a tile. P goes back to TMEM as the A operand of the value product, in the place
// of its half's scores, instead of through shared memory. A tile takes 1,800 cycles, so that head
// dims of 128 run at the memory's pace where a unit is one row block, and head dim 64, or several row
// blocks per KV head, at the softmax's: 16 traces x 4,096 rows, 8 KV heads, R = 128, head dim 128 / 64
// 45 / 42 us; 4 traces x 4,096 rows, 4 KV heads, R = 512 31 us. With keys on the lanes the same tile took
// 3,500 cycles (tables of references and sums per thread, P and both operand streams through shared
// memory). What did not help: two groups of four warps on alternate tiles, 128 scores a thread (the
// same times for long runs of tiles, 10 % longer ones for short units); an eighth or a quarter of
// the exponentials as polynomials (nothing, 4 % longer); turns at the exponentials for the two warps
// of a row (tiles of 1,480 cycles, the same times).
// ---------------------------------------------------------------------------
constexpr int kRowsThreads = 256 + 96;  // softmax, TMA, score products, value products

// 32 consecutive TMEM columns of packed pairs
__device__ __forceinline__ void tc_st32(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}

// A from TMEM
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.u32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "n"(kDescHigh)
      : "memory");
}

// Two fp32 operations in one instruction, and the largest of three.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\t"
      "mov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int PANELS, bool BF16>
__global__ void __launch_bounds__(kRowsThreads, 1) k_tree_attn_rows(const __grid_constant__ TreeMmaParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int DP = PANELS * 64;
  constexpr int kSoft = 256;
  constexpr uint32_t kO = 2 * kTile;  // TMEM columns: scores of two tiles, then an O of either half of the keys
  const TreeSmem lay = tree_smem(PANELS, p.n16, p.nst, p.nq);
  uint8_t* misc = smem + lay.misc;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(misc);
  uint64_t* kv_empty = kv_full + kMaxStages;
  uint64_t* s_full = kv_empty + kMaxStages;  // [2]
  uint64_t* q_full = s_full + 2;             // [2]
  uint64_t* q_empty = q_full + 2;            // [2]
  uint64_t* p_full = q_empty + 2;            // [2 halves][2]
  uint64_t* pv_done = p_full + 4;            // [2]
  uint64_t* o_empty = pv_done + 2;
  const TreeBars bars = {kv_full, kv_empty, q_full, q_empty};
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(o_empty + 1);
  float2* xchg = reinterpret_cast<float2*>(misc + kMiscRef);  // [128] between the two threads of a row
  TraceTable& tab = *reinterpret_cast<TraceTable*>(misc + kMiscTab);
  volatile uint32_t* noted = reinterpret_cast<uint32_t*>(misc + kMiscNoted);  // drafted rows of two segments

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TreeAttnArgs& a = p.a;
  const int R = p.mb * p.G;
  bool dead = false;

  if (warp == 8) {
    if (lane < 7) prefetch_map(&p.mq + lane);
    if (lane == 0) {
      for (int i = 0; i < kMaxStages; ++i) {
        mbar_init(kv_full + i, 1);
        mbar_init(kv_empty + i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + i, 1);
        mbar_init(q_full + i, 1);
        mbar_init(q_empty + i, 1);
        mbar_init(p_full + i, kSoft / 2);
        mbar_init(p_full + 2 + i, kSoft / 2);
        mbar_init(pv_done + i, 1);
      }
      mbar_init(o_empty, kSoft);
      fence_mbar_init();
    }
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_base), 512);
  } else {
    zero_query_tail(smem + lay.q, PANELS * p.nq, p.n16, R, tid, kSoft);
  }
  pdl_wait();
  pdl_launch_dependents();
  tc_before_sync();
  if (warp == 8) {
    prefix_tiles(p, tab, lane, a.Hkv * p.RB);
    __syncwarp();
    asm volatile("bar.arrive 9, %0;" ::"n"(kRowsThreads) : "memory");
  } else {
    named_bar_sync(9, kRowsThreads);
  }
  tc_after_sync();
  const int c = blockIdx.x;
  int beg, end;
  cta_share(p, tab, c, &beg, &end);
  const uint32_t ring = smem_u32(smem + lay.ring), qbase = smem_u32(smem + lay.q);

  if (warp == 8) {
    tma_role<PANELS>(p, tab, lay, bars, beg, end, ring, qbase, R);
  } else if (warp == 9) {
    // ---------------------------------------------------------------- scores
    const uint32_t idesc = instr_desc(BF16, kTile, false, false);
    const uint32_t ring_k = smem_desc(ring, 16), q_desc = smem_desc(qbase, 16);
    const uint32_t tmem = *tmem_base;
    int k = 0, seg = 0, st = 0, use = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, p.RB, s); ++seg) {
      const int qs = p.nq == 2 ? seg & 1 : 0, quse = p.nq == 2 ? seg >> 1 : seg;
      guarded_wait(q_full + qs, quse & 1, dead, a.err);
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        guarded_wait(kv_full + st, use & 1, dead, a.err);
        // the buffer of tile k - 2 holds its P until its value product has read it
        if (k >= 2) guarded_wait(pv_done + (k & 1), ((k >> 1) - 1) & 1, dead, a.err);
        tc_after_sync();
        if (elect_one()) {
          const uint32_t ka = ring_k + (st * lay.stage >> 4), qa = q_desc + (qs * lay.qslot >> 4);
#pragma unroll
          for (int kk = 0; kk < PANELS * 4; ++kk)
            tc_mma(tmem + (k & 1) * kTile, qa + (kk >> 2) * (kPanel >> 4) + (kk & 3) * 2,
                   ka + (kk >> 2) * (kPanel >> 4) + (kk & 3) * 2, idesc, kk > 0);
          tc_commit(s_full + (k & 1));
          tc_commit(kv_empty + st);
          if (jj + 1 == s.n) tc_commit(q_empty + qs);
        }
        __syncwarp();
        next_tile(p.nst, st, use);
      }
    }
    if (dead) drain_products();
  } else if (warp == 10) {
    // ---------------------------------------------------------------- values
    const uint32_t idesc = instr_desc(BF16, DP, false, true);
    const uint32_t ring_v = smem_desc(ring, kPanel);
    const uint32_t tmem = *tmem_base;
    int k = 0, seg = 0, st = 1, use = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, p.RB, s); ++seg) {
      const SegmentMasks masks = load_masks(a, s.t, lane);
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        const bool draft = s.j0 + jj == s.nt - 1;
        const int rows = tile_rows(s.len, s.nt, a.m, s.j0 + jj), steps = (rows + 15) / 16;
        guarded_wait(kv_full + st, use & 1, dead, a.err);
        if (rows & 15 || draft)
          prepare_values<PANELS, BF16>(smem + lay.ring + st * lay.stage, rows, draft, masks, lane, noted + 2 * (seg & 1));
        if (jj == 0 && seg >= 1) guarded_wait(o_empty, (seg - 1) & 1, dead, a.err);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          guarded_wait(p_full + 2 * half + (k & 1), (k >> 1) & 1, dead, a.err);
          tc_after_sync();
          if (elect_one()) {
            const uint32_t va = ring_v + (st * lay.stage >> 4) + half * (8192 >> 4);
            const uint32_t pa = tmem + (k & 1) * kTile + half * 64, o = tmem + kO + half * DP;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (half * 4 + kk < steps) tc_mma_ts(o, pa + kk * 8, va + kk * (2048 >> 4), idesc, jj > 0 || kk > 0);
            if (half == 1) {
              tc_commit(kv_empty + st);
              tc_commit(pv_done + (k & 1));
            }
          }
          __syncwarp();
        }
        __syncwarp();
        next_tile(p.nst, st, use);
      }
    }
    if (dead) drain_products();
  } else {
    // ---------------------------------------------------------------- softmax
    const int grp = warp >> 2, wq = warp & 3;
    const int row = wq * 32 + lane;  // this thread's row; keys 64 grp .. 64 grp + 63 of a tile
    const int key0 = 64 * grp;
    const bool idle = wq * 32 >= R;  // no row of the warp is real
    const uint32_t tmem = *tmem_base, lanes = static_cast<uint32_t>(wq * 32) << 16;
    const float sc = a.scale_log2;
    const int my_node = row / p.G, my_head = row - my_node * p.G;
    auto stage_piece = [&](int r, int q) {  // 16 bytes of row r's line in the warp's 2 KB
      return reinterpret_cast<uint4*>(smem + lay.p + warp * 2048 + r * 64 + ((q ^ (r >> 1)) & 3) * 16);
    };
    int seg = 0, k = 0;
    Segment s, next;
    uint64_t mask = 0, next_mask = 0;  // of this row
    int f = beg;
    bool more = next_segment(p, tab, f, end, p.RB, s);
    auto mask_of = [&](const Segment& g) {
      const int node = g.rb * p.mb + my_node;
      return row < R && node < a.m ? ld_mask(a.masks + g.t * a.mask_stride + node) : 0;
    };
    if (more) mask = mask_of(s);
    for (; more; ++seg, s = next, mask = next_mask) {
      const int node = s.rb * p.mb + my_node;
      const bool real_row = row < R && node < a.m;
      const uint32_t obuf = tmem + lanes + kO;
      float ref = kNoRef, l = 0.0f;
      for (int jj = 0; jj < s.n; ++jj, ++k) {
        const int j = s.j0 + jj;
        const bool draft = j == s.nt - 1;
        const int rows = tile_rows(s.len, s.nt, a.m, j);
        const uint32_t sbuf = tmem + lanes + (k & 1) * kTile;
        guarded_wait(s_full + (k & 1), (k >> 1) & 1, dead, a.err);
        tc_after_sync();
        if (idle || rows <= key0) {  // nothing of this half is used
          mbar_arrive(p_full + 2 * grp + (k & 1));
          continue;
        }
        float x[64];
#pragma unroll
        for (int i = 0; i < 64; i += 16) tc_ld16(sbuf + key0 + i, x + i);
        tc_wait_ld();
        // scores are x * f: f is the scale, or 1 where the scale is applied with the mask. For a
        // negative scale the products change sign first, so that the largest x is the largest score.
        float f = fabsf(sc);
        if (sc < 0.0f) {
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = -x[i];
        }
        if (draft || rows < kTile) {
          // bits of this thread's 64 keys that the row sees
          uint64_t see = draft ? (grp == 0 ? mask : 0) : ~0ull;
          const int n = rows - key0;  // valid keys among them
          see &= n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
          const uint32_t lo = static_cast<uint32_t>(see), hi = static_cast<uint32_t>(see >> 32);
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            const bool on = ((i < 32 ? lo : hi) >> (i & 31)) & 1;
            x[i] = on ? x[i] * f : -INFINITY;
          }
          f = 1.0f;
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) top[u] = max3(top[u], x[i + u], x[i + u + 4]);
        }
        const float mx = max3(top[0], top[1], fmaxf(top[2], top[3])) * f;
        if (__any_sync(0xffffffffu, mx > ref + kSlack)) {
          const float now = fmaxf(mx, ref), fade = ex2(ref - now);
          ref = now;
          l *= fade;
          if (jj > 0) {  // O as the last product left it
            guarded_wait(pv_done + ((k - 1) & 1), ((k - 1) >> 1) & 1, dead, a.err);
            tc_after_sync();
#pragma unroll 1
            for (int i = 0; i < DP; i += 16) {
              float o[16];
              tc_ld16(obuf + grp * DP + i, o);
              tc_wait_ld();
#pragma unroll
              for (int u = 0; u < 16; ++u) o[u] *= fade;
              tc_st16(obuf + grp * DP + i, o);
            }
          }
        }
        // p = 2^(x - m_ref), one rounding to the inputs' type for the product with V
        uint32_t pk[32];
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        const float2 f2 = make_float2(f, f), ref2 = make_float2(-ref, -ref);
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float2 e = fma2(make_float2(x[i], x[i + 1]), f2, ref2);
          e.x = ex2(e.x);
          e.y = ex2(e.y);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
          pk[i / 2] = pack2<BF16>(e.x, e.y);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tc_st32(sbuf + key0, pk);  // in the place of this half's scores
        tc_wait_st();
        tc_before_sync();
        mbar_arrive(p_full + 2 * grp + (k & 1));
      }
      // ------------------------------------------------ end of the segment: sums, output
      more = next_segment(p, tab, f, end, p.RB, next);  // under the last value product
      if (more) next_mask = mask_of(next);
      // The two halves' parts of a row: the second hands over its reference and sum and gets the
      // factors for the two O. Without a tile of more than 64 keys nothing valid is in the second's
      // (such a tile is the segment's first or there is none).
      const bool has1 = tile_rows(s.len, s.nt, a.m, s.j0) > 64, whole = s.n == s.nt;
      const int slot = 2 * c + (s.j0 > 0 ? 0 : 1);
      float2 fac;
      if (grp == 1) xchg[row] = make_float2(ref, l);
      named_bar_sync(1 + wq, 64);
      if (grp == 0) {
        const float2 other = xchg[row];
        const float both = fmaxf(ref, other.x);
        fac = make_float2(ex2(ref - both), ex2(other.x - both));
        const float sum = l * fac.x + other.y * fac.y;
        const bool some = mask != 0 && sum != 0.0f;
        if (!whole) {
          float* ml = p.ml + static_cast<int64_t>(slot) * 2 * kMaxRows;
          ml[row] = both;
          ml[kMaxRows + row] = some ? sum : 0.0f;
        } else {
          if (p.lse) {
            const int64_t unit = (static_cast<int64_t>(s.t) * a.Hkv + s.kvh) * p.RB + s.rb;
            p.lse[unit * kMaxRows + row] = some ? both + log2f(sum) : INFINITY;
          }
          const float inv = some ? 1.0f / sum : 0.0f;
          fac = make_float2(some ? fac.x * inv : -1.0f, fac.y * inv);  // -1: a row without keys
        }
        xchg[row] = fac;
      }
      named_bar_sync(1 + wq, 64);
      if (grp == 1) fac = xchg[row];
      const bool real = !(fac.x < 0.0f);
      uint16_t* out =
          real_row ? a.out + s.t * a.os[0] + node * a.os[1] + (s.kvh * p.G + my_head) * a.os[2] : nullptr;
      float* part = p.part + (static_cast<int64_t>(slot) * R + wq * 32) * DP;  // of the warp's rows
      guarded_wait(pv_done + ((k - 1) & 1), ((k - 1) >> 1) & 1, dead, a.err);
      tc_after_sync();
      const volatile uint32_t* nt = noted + 2 * (seg & 1);
      const uint64_t bad = s.j0 + s.n == s.nt ? mask & (static_cast<uint64_t>(nt[1]) << 32 | nt[0]) : 0;
#pragma unroll 1
      for (int i = grp * (DP / 2); i < (grp + 1) * (DP / 2); i += 16) {
        float o[16], o1[16];
        tc_ld16(obuf + i, o);
        tc_ld16(obuf + DP + i, o1);
        tc_wait_ld();
#pragma unroll
        for (int u = 0; u < 16; ++u) o[u] = o[u] * fac.x + (has1 ? o1[u] * fac.y : 0.0f);
        // Through shared memory, so that a store writes 64 bytes of a row, not 16: a line of 64
        // bytes per row, its pieces swizzled.
        if (!whole) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *stage_piece(lane, q) = make_uint4(__float_as_uint(o[4 * q]), __float_as_uint(o[4 * q + 1]),
                                               __float_as_uint(o[4 * q + 2]), __float_as_uint(o[4 * q + 3]));
          __syncwarp();
          uint4 y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = *stage_piece(8 * u + (lane >> 2), lane & 3);
          float* to = part + (lane >> 2) * DP + i + (lane & 3) * 4;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (8 * u + (lane >> 2) < R - wq * 32) *reinterpret_cast<uint4*>(to + 8 * u * DP) = y[u];
          __syncwarp();
        } else {
          const int half = (i >> 4) & 1;  // 32 columns at a time
          uint32_t w[8];
#pragma unroll
          for (int u = 0; u < 16; u += 2) w[u / 2] = real ? pack2<BF16>(o[u], o[u + 1]) : 0u;
          *stage_piece(lane, 2 * half) = make_uint4(w[0], w[1], w[2], w[3]);
          *stage_piece(lane, 2 * half + 1) = make_uint4(w[4], w[5], w[6], w[7]);
          if (half) {
            __syncwarp();
            const int col = i - 16 + (lane & 3) * 8;  // the head dim is a multiple of 8
            uint4 y[4];
            unsigned long long to[4];  // of the four rows, 0 if there is none
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              y[u] = *stage_piece(8 * u + (lane >> 2), lane & 3);
              to[u] = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), 8 * u + (lane >> 2));
            }
            if (col < a.d && p.vec_out) {
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (to[u]) *reinterpret_cast<uint4*>(to[u] + 2 * col) = y[u];
            } else if (col < a.d) {
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                if (!to[u]) continue;
                uint16_t* o16 = reinterpret_cast<uint16_t*>(to[u]) + col;
                const uint32_t z[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                  o16[2 * v] = static_cast<uint16_t>(z[v]);
                  o16[2 * v + 1] = static_cast<uint16_t>(z[v] >> 16);
                }
              }
            }
            __syncwarp();
          }
        }
      }
      if (__any_sync(0xffffffffu, bad != 0)) {  // rare; after the warp's stores
        __syncwarp();
        const int c0 = grp * (DP / 2), c1 = min(a.d, c0 + DP / 2);
        if (bad && !whole)
          add_noted<BF16>(a, s.t, s.kvh, bad, nullptr, part + lane * DP, c0, c1);
        else if (bad && real)
          add_noted<BF16>(a, s.t, s.kvh, bad, out, nullptr, c0, c1);
      }
      tc_before_sync();
      mbar_arrive(o_empty);
    }
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (warp == 9) tmem_dealloc(*tmem_base, 512);
}

// Joins the pieces of the units that were cut between CTAs, in order: CTA (x, y) a group of the rows
// of unit x (join_by_unit) or of the unit whose first cut lies at boundary x between attention CTAs.
// Where the cuts lie it works out from the lengths, which it may read before
// the attention has finished (that began only after the kernels that wrote them had), so that one
// round of loads is left after the wait. One CTA per unit and 8 rows, most with nothing to join,
// took 6 us after a 17 us attention; notes left by the attention, read after the wait, 1 to 2.5 us
// more than this where the units are few.
constexpr int kJoinBlock = 256;

template <int PANELS, bool BF16>
__global__ void __launch_bounds__(kJoinBlock) k_tree_join(const __grid_constant__ TreeMmaParams p) {
  constexpr int DP = PANELS * 64;
  constexpr int kLanes = DP / 4;  // threads of a row, four values each
  __shared__ TraceTable tab;
  const int tid = threadIdx.x;
  const TreeAttnArgs& a = p.a;
  pdl_launch_dependents();  // the weight pass loads its keys meanwhile
  // Without a unit to join. What comes after this grid waits for it alone, so it must not complete
  // before the attention has: its first CTA stays until then (all of them: trees of 63 25.1 us, 24.7 so).
  auto leave = [] {
    if (blockIdx.x == 0 && blockIdx.y == 0) pdl_wait();
  };
  const int units = a.Hkv * p.RB;
  if (tid < 32) prefix_tiles(p, tab, tid, units);
  __syncthreads();
  const int total = tab.cum[p.T], g = min(p.grid, total);
  if (share_mode(p, total, tab.max_span, units * p.T) != Share::kCut) return leave();
  int lo, u, c0;
  if (p.join_by_unit) {
    lo = blockIdx.x / units;
    u = blockIdx.x - lo * units;
  } else {
    c0 = blockIdx.x;
    if (c0 + 1 >= g) return leave();
    const int here = cut(total, c0 + 1, g);
    lo = 0;
    int hi = p.T - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (tab.cum[mid] <= here)
        lo = mid;
      else
        hi = mid - 1;
    }
    u = (here - tab.cum[lo]) / unit_span(trace_tiles(tab.len[lo]));
  }
  const int nt = trace_tiles(tab.len[lo]), tile0 = tab.cum[lo] + u * unit_span(nt) + kUnitCost;
  // its first and its last piece: the largest c with cut(c) <= the position of a tile
  const int first = static_cast<int>((static_cast<int64_t>(tile0 + 1) * g - 1) / total);
  const int c1 = static_cast<int>((static_cast<int64_t>(tile0 + nt) * g - 1) / total);
  if (first == c1 || (!p.join_by_unit && first != c0)) return leave();  // whole, or first cut elsewhere
  c0 = first;
  const int tr = p.t0 + lo, kvh = u / p.RB, rb = u - kvh * p.RB;
  const int R = p.mb * p.G, v = (tid % kLanes) * 4;
  int n = blockIdx.y * p.join_passes * (kJoinBlock / kLanes) + tid / kLanes;
  pdl_wait();
  for (int pass = 0; pass < p.join_passes; ++pass, n += kJoinBlock / kLanes) {
    const int node = rb * p.mb + n / p.G;
    if (n >= R || node >= a.m) break;
    const bool shown = a.masks[tr * a.mask_stride + node] != 0;
    float top = kNoRef, sum = 0.0f, o[4] = {};
    for (int b = c0; b <= c1; b += 4) {  // four pieces' loads in flight, one round of latency for most units
      float m[4], l[4];
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + i <= c1) {
          const int64_t slot = 2 * (b + i) + (b + i == c0 ? 1 : 0);
          m[i] = p.ml[slot * 2 * kMaxRows + n];
          l[i] = p.ml[(slot * 2 + 1) * kMaxRows + n];
          x[i] = *reinterpret_cast<const float4*>(p.part + (slot * R + n) * DP + v);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + i <= c1) {
          const float now = fmaxf(top, m[i]), fade = ex2(top - now), w = ex2(m[i] - now);
          top = now;
          sum = fmaf(w, l[i], sum * fade);
          o[0] = fmaf(w, x[i].x, o[0] * fade);
          o[1] = fmaf(w, x[i].y, o[1] * fade);
          o[2] = fmaf(w, x[i].z, o[2] * fade);
          o[3] = fmaf(w, x[i].w, o[3] * fade);
        }
    }
    const bool real = shown && sum != 0.0f;
    const float inv = real ? 1.0f / sum : 0.0f;
    uint16_t* out = a.out + tr * a.os[0] + node * a.os[1] + (kvh * p.G + n % p.G) * a.os[2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v + i < a.d) out[v + i] = round16<BF16>(real ? o[i] * inv : 0.0f);
    if (p.lse && v == 0)
      p.lse[((static_cast<int64_t>(tr) * a.Hkv + kvh) * p.RB + rb) * kMaxRows + n] =
          real ? top + log2f(sum) : INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Attention weight of every row, summed over the nodes and heads that read it:
//   w_l = sum_rows 2^(x_l - lse_row),  x = scale log2(e) q . k.
// The row maxima are known only when all keys have been seen, so the scores are formed again
// (K once more through the same ring and product; V is not needed) and a thread, which holds
// one key, adds over the rows of its lane: no exchange between threads. Row blocks follow one
// another within a CTA, and a row's sum is always kept by the same thread.
// ---------------------------------------------------------------------------
constexpr int kWeightThreads = 256 + 64;

template <int PANELS, bool BF16>
__global__ void __launch_bounds__(kWeightThreads, 1) k_tree_weights(const __grid_constant__ TreeMmaParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kSoft = 256;  // two warpgroups take alternate tiles
  const TreeSmem lay = tree_smem(PANELS, p.n16, p.nst, p.nq);
  uint8_t* misc = smem + lay.misc;
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(misc);
  uint64_t* kv_empty = kv_full + kMaxStages;
  uint64_t* s_full = kv_empty + kMaxStages;
  uint64_t* s_empty = s_full + 2;
  uint64_t* q_full = s_empty + 2;
  uint64_t* q_empty = q_full + 2;
  uint32_t* tmem_base = reinterpret_cast<uint32_t*>(q_empty + 2);
  TraceTable& tab = *reinterpret_cast<TraceTable*>(misc + kMiscTab);
  // per warpgroup the rows' lse and draft masks, and a bit per row that sees anything: in the last
  // ring stage, which is left out
  float* lse_s = reinterpret_cast<float*>(smem + lay.ring + (p.nst - 1) * lay.stage);
  uint64_t* mask_s = reinterpret_cast<uint64_t*>(lse_s + 2 * kMaxRows);
  uint32_t* live_s = reinterpret_cast<uint32_t*>(mask_s + 2 * kMaxRows);
  const int nst = p.nst - 1;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const TreeAttnArgs& a = p.a;
  const int R = p.mb * p.G;
  bool dead = false;
  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < kMaxStages; ++i) {
        mbar_init(kv_full + i, 1);
        mbar_init(kv_empty + i, 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + i, 1);
        mbar_init(s_empty + i, 128);
        mbar_init(q_full + i, 1);
        mbar_init(q_empty + i, 1);
      }
      fence_mbar_init();
    }
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_base), 256);
  } else {
    zero_query_tail(smem + lay.q, PANELS * p.nq, p.n16, R, tid, kSoft);
  }
  // Lengths, queries, keys and masks were written before the attention began, so the TMA and MMA
  // warps do not wait for the join: the first score products are ready when its results are.
  tc_before_sync();
  if (warp == 8) {
    prefix_tiles(p, tab, lane, a.Hkv);  // units are (trace, KV head) here: the sequence has no row blocks
    __syncwarp();
    asm volatile("bar.arrive 3, %0;" ::"n"(kWeightThreads) : "memory");
  } else {
    named_bar_sync(3, kWeightThreads);
  }
  tc_after_sync();
  const int total = tab.cum[p.T];
  const int g = min(p.grid, total);
  const int c = blockIdx.x;
  const int beg = c < g ? cut(total, c, g) : 0, end = c < g ? cut(total, c + 1, g) : 0;
  const uint32_t ring = smem_u32(smem + lay.ring), qbase = smem_u32(smem + lay.q);

  if (warp == 8) {
    const uint64_t policy = policy_evict_first(), keep = policy_evict_last();
    int item = 0, seg = 0, st = 0, use = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, 1, s);) {
      for (int rb = 0; rb < p.RB; ++rb, ++seg) {
        const int qs = p.nq == 2 ? seg & 1 : 0, quse = p.nq == 2 ? seg >> 1 : seg;
        const uint64_t pol = rb + 1 < p.RB ? keep : policy;
        for (int j = s.j0; j < s.j0 + s.n; ++j, ++item) {
          const int rows = tile_rows(s.len, s.nt, a.m, j);
          if (use > 0) guarded_wait(kv_empty + st, (use - 1) & 1, dead, a.err);
          const uint32_t dst = ring + st * lay.stage;
          if (elect_one()) {
            if (j == s.nt - 1) {
              mbar_expect_tx(kv_full + st, PANELS * 128 * a.m);
              for (int pn = 0; pn < PANELS; ++pn)
                tma_load_4d(dst + pn * kPanel, &p.mkd, kv_full + st, pn * 64, s.kvh, 0, s.t, keep);
            } else if (rows == kTile) {
              mbar_expect_tx(kv_full + st, PANELS * kPanel);
              for (int pn = 0; pn < PANELS; ++pn)
                tma_load_4d(dst + pn * kPanel, &p.mk, kv_full + st, pn * 64, j * kTile, s.kvh, s.t, pol);
            } else {
              const int boxes = (rows + kBox - 1) / kBox;
              mbar_expect_tx(kv_full + st, PANELS * 128 * boxes * kBox);
              for (int pn = 0; pn < PANELS; ++pn)
                for (int b = 0; b < boxes; ++b)
                  tma_load_4d(dst + pn * kPanel + b * kBox * 128, &p.mk_end, kv_full + st, pn * 64,
                              j * kTile + b * kBox, s.kvh, s.t, pol);
            }
          }
          __syncwarp();
          if (++st == nst) {
            st = 0;
            ++use;
          }
          if (j == s.j0) {
            if (quse > 0) guarded_wait(q_empty + qs, (quse - 1) & 1, dead, a.err);
            if (elect_one()) {
              mbar_expect_tx(q_full + qs, PANELS * R * 128);
              for (int pn = 0; pn < PANELS; ++pn)
                tma_load_4d(qbase + qs * lay.qslot + pn * p.n16 * 128, &p.mq, q_full + qs, pn * 64, s.kvh * p.G,
                            rb * p.mb, s.t, keep);
            }
            __syncwarp();
          }
        }
      }
    }
    if (dead)
      for (int i = max(0, item - nst); i < item; ++i) mbar_wait(kv_full + i % nst, (i / nst) & 1);
  } else if (warp == 9) {
    const uint32_t id_qk = instr_desc(BF16, p.used, false, false);
    const uint32_t ring_k = smem_desc(ring, 16), q_desc = smem_desc(qbase, 16);
    const uint32_t qpanel = p.n16 * 128 >> 4;
    const uint32_t tmem = *tmem_base;
    int seg = 0, st = 0, use = 0, fills0 = 0, fills1 = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, 1, s);) {
      for (int rb = 0; rb < p.RB; ++rb, ++seg) {
        const int qs = p.nq == 2 ? seg & 1 : 0, quse = p.nq == 2 ? seg >> 1 : seg;
        guarded_wait(q_full + qs, quse & 1, dead, a.err);
        for (int jj = 0; jj < s.n; ++jj) {
          guarded_wait(kv_full + st, use & 1, dead, a.err);
          // buffer b belongs to warpgroup b, which waits for every one of its fills
          const int b = jj & 1, fill = b ? fills1++ : fills0++;
          if (fill > 0) guarded_wait(s_empty + b, (fill - 1) & 1, dead, a.err);
          tc_after_sync();
          if (elect_one()) {
            const uint32_t ka = ring_k + (st * lay.stage >> 4), qb = q_desc + (qs * lay.qslot >> 4);
#pragma unroll
            for (int kk = 0; kk < PANELS * 4; ++kk)
              tc_mma(tmem + b * kMaxRows, ka + (kk >> 2) * (kPanel >> 4) + (kk & 3) * 2,
                     qb + (kk >> 2) * qpanel + (kk & 3) * 2, id_qk, kk > 0);
            tc_commit(s_full + b);
            tc_commit(kv_empty + st);
            if (jj + 1 == s.n) tc_commit(q_empty + qs);
          }
          __syncwarp();
          if (++st == nst) {
            st = 0;
            ++use;
          }
        }
      }
    }
    if (dead) drain_products();
  } else {
    const int grp = warp >> 2, wq = warp & 3;
    const int key = wq * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(wq * 32) << 16;
    const float sc = a.scale_log2;
    float* lse = lse_s + grp * kMaxRows;
    uint64_t* rowmask = mask_s + grp * kMaxRows;
    uint32_t* live = live_s + grp * (kMaxRows / 32);
    const uint32_t sbuf = *tmem_base + lanes + grp * kMaxRows;
    pdl_wait();  // the join's denominators
    pdl_launch_dependents();
    int fill = 0;
    Segment s;
    for (int f = beg; next_segment(p, tab, f, end, 1, s);) {
      const int64_t unit = static_cast<int64_t>(s.t) * a.Hkv + s.kvh;
      for (int rb = 0; rb < p.RB; ++rb) {
        named_bar_sync(1 + grp, 128);  // the last block's tables read
        const int i = rb * p.mb + key / p.G;
        const bool node = key < R && i < a.m;  // the last block may hold fewer nodes
        const float norm = node ? p.lse[(unit * p.RB + rb) * kMaxRows + key] : INFINITY;
        lse[key] = norm;
        rowmask[key] = node ? a.masks[s.t * a.mask_stride + i] : 0;
        const uint32_t seeing = __ballot_sync(0xffffffffu, norm != INFINITY);
        if (lane == 0) live[wq] = seeing;
        named_bar_sync(1 + grp, 128);
        bool all_live = true;
        for (int n = 0; n < p.used; n += 16) all_live &= (live[n >> 5] >> (n & 16) & 0xFFFFu) == 0xFFFFu;
        for (int jj = grp; jj < s.n; jj += 2, ++fill) {
          const int j = s.j0 + jj;
          const bool draft = j == s.nt - 1;
          const int rows = tile_rows(s.len, s.nt, a.m, j);
          guarded_wait(s_full + grp, fill & 1, dead, a.err);
          tc_after_sync();
          // Rows that see nothing (padding nodes, the block's tail) are left out by their bits: their
          // scores may be anything, and 2^(x - inf) is 0 only for an x that is a number below inf.
          // Measured, 4 traces of 16 nodes, one padded: 36.7 us (without the test 36.2, with a condition
          // per row, which becomes a branch, in place of the & 37.2).
          float w = 0.0f, x[16], ls[16];
          auto add = [&](int n, auto weigh) {
            load16(lse + n, ls);
            tc_ld16(sbuf + n, x);
            tc_wait_ld();
            float part = 0.0f;
#pragma unroll
            for (int u = 0; u < 16; ++u) part += weigh(u, ex2(fmaf(x[u], sc, -ls[u])));
            w += part;
          };
          if (draft) {
            for (int n = 0; n < p.used; n += 16)
              add(n, [&](int u, float e) { return (rowmask[n + u] >> (key & 63)) & 1 ? e : 0.0f; });
          } else if (all_live) {
            for (int n = 0; n < p.used; n += 16) add(n, [](int, float e) { return e; });
          } else {
            for (int n = 0; n < p.used; n += 16) {
              const uint32_t on = live[n >> 5] >> (n & 16) & 0xFFFFu;
              if (on != 0)
                add(n, [&](int u, float e) { return __uint_as_float(__float_as_uint(e) & (0u - ((on >> u) & 1u))); });
            }
          }
          tc_before_sync();
          mbar_arrive(s_empty + grp);
          if (key < rows) {
            float* dst = draft ? a.draft_scores + unit * a.m + key : a.scores_out + unit * a.Lmax + j * kTile + key;
            const float base = rb > 0 ? *dst : draft || !a.scores ? 0.0f : a.scores[unit * a.Lmax + j * kTile + key];
            *dst = base + w;
          }
        }
      }
    }
  }
  tc_before_sync();
  __syncthreads();
  tc_after_sync();
  if (warp == 9) tmem_dealloc(*tmem_base, 256);
}

// The same sums where the attention kept its scores (few rows): a thread per four cached rows.
// R reads of four bytes per row instead of 2 d bytes of its key.
constexpr int kKeptBlock = 128;

__global__ void __launch_bounds__(kKeptBlock) k_tree_weights_kept(const __grid_constant__ TreeMmaParams p) {
  __shared__ float lse[kKeysRows];
  __shared__ uint64_t see[kKeysRows];  // drafted rows
  pdl_wait();
  pdl_launch_dependents();
  const TreeAttnArgs& a = p.a;
  const int R = p.mb * p.G, tid = threadIdx.x;
  const int t = p.t0 + blockIdx.y / a.Hkv;
  const int64_t unit = static_cast<int64_t>(p.t0) * a.Hkv + blockIdx.y;
  const int len = trace_len(a, t), l0 = (blockIdx.x * kKeptBlock + tid) * 4;
  if (blockIdx.x * kKeptBlock * 4 >= len && blockIdx.x > 0) return;
  if (tid < R) {
    lse[tid] = p.lse[unit * kMaxRows + tid];
    see[tid] = a.masks[t * a.mask_stride + tid / p.G];
  }
  __syncthreads();
  if (l0 < len) {
    float w[4] = {};
    const float* x = p.kept + unit * R * p.kept_len + l0;
    for (int r = 0; r < R; ++r) {
      if (lse[r] == INFINITY) continue;  // a row that sees nothing: its scores may be anything
      const float4 v = *reinterpret_cast<const float4*>(x + static_cast<int64_t>(r) * p.kept_len);
      w[0] += ex2(v.x - lse[r]);
      w[1] += ex2(v.y - lse[r]);
      w[2] += ex2(v.z - lse[r]);
      w[3] += ex2(v.w - lse[r]);
    }
    const int64_t at = unit * a.Lmax + l0;
    for (int i = 0; i < 4 && l0 + i < len; ++i) a.scores_out[at + i] = (a.scores ? a.scores[at + i] : 0.0f) + w[i];
  }
  if (blockIdx.x == 0 && tid < a.m) {
    float w = 0.0f;
    for (int r = 0; r < R; ++r)  // by the masks: the kept -inf of a row that is not seen, less an lse of NaN, is NaN
      if ((see[r] >> tid) & 1) w += ex2(p.kept_draft[(unit * R + r) * 64 + tid] - lse[r]);
    a.draft_scores[unit * a.m + tid] = w;
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Caches this short are not cut, whatever their lengths: a CTA does its whole unit and no join is
// launched. Measured: 16 units of 203 rows 6.8 us (7.1 with a join that finds nothing to do), 144 units
// of 100 to 500 rows 9.0 us (9.7).
constexpr int kWholeRows = 512;

struct TreePlan {
  int G, RB, mb, n16, used, panels, nst, nq, grid;
  uint32_t smem;
};

static bool tree_plan(int T, int m, int H, int Hkv, int Lmax, int d, TreePlan* pl) {
  pl->G = H / Hkv;
  if (pl->G > kMaxRows || d > 128 || d % 8 != 0) return false;
  const int fit = kMaxRows / pl->G;  // nodes of a full block
  pl->RB = (m + fit - 1) / fit;
  pl->mb = (m + pl->RB - 1) / pl->RB;  // even blocks
  pl->RB = (m + pl->mb - 1) / pl->mb;
  pl->n16 = (pl->mb * pl->G + 15) / 16 * 16;
  pl->used = pl->n16;
  if (pl->n16 > kKeysRows) pl->n16 = kMaxRows;  // k_tree_attn_rows: rows fill the lanes
  pl->panels = d > 64 ? 2 : 1;
  pl->grid = sm_count();
  // flat tile numbers are 32-bit
  if (static_cast<int64_t>(std::min(T, kMaxTraces)) * Hkv * pl->RB * (Lmax / kTile + 2) > 0x7FFFFFFFll) return false;
  // two Q slots (the next unit's queries load early) where they leave a ring of five stages
  const uint32_t cap = 227 * 1024;
  for (pl->nq = 2;; --pl->nq) {
    const uint32_t fixed = tree_smem(pl->panels, pl->n16, 0, pl->nq).total;
    pl->nst = std::min<int>(kMaxStages, (cap - fixed) / (pl->panels * kPanel));
    if (pl->nst >= 5 || pl->nq == 1) break;
  }
  pl->smem = tree_smem(pl->panels, pl->n16, pl->nst, pl->nq).total;
  return pl->nst >= 4;
}

// Rows whose scores are kept for the weight pass rather than formed again from K: 8 R bytes of
// workspace traffic per key instead of 2 d. Measured, 256 units of 4,096 rows of 128: R = 1 90.7 us
// (123.7 formed again), R = 8 97.8 (125.7), R = 16 114.0 (127.3); head dim 64, R = 16 alike.
constexpr int kKeptRows = kKeysRows;

size_t tree_mma_workspace(int T, int m, int H, int Hkv, int Lmax, int d, bool with_scores) {
  TreePlan pl;
  if (!tree_plan(T, m, H, Hkv, Lmax, d, &pl)) return 0;
  const size_t part = static_cast<size_t>(2) * pl.grid * pl.mb * pl.G * pl.panels * 64 * 4;
  const size_t ml = static_cast<size_t>(2) * pl.grid * 2 * kMaxRows * 4;
  if (!with_scores) return part + ml + 256;
  const size_t lse = static_cast<size_t>(T) * Hkv * pl.RB * kMaxRows * 4;
  const int R = pl.mb * pl.G;
  const size_t kept = R <= kKeptRows ? static_cast<size_t>(T) * Hkv * R * ((Lmax + 3) / 4 * 4 + 64) * 4 : 0;
  return part + ml + lse + kept + 256;
}

bool tree_mma_takes(const TreeAttnArgs& a) {
  // tensor maps: 16-byte bases, positive strides in multiples of 16 bytes below 2^40
  const struct {
    const void* p;
    const int64_t* s;
    int n[3];
  } t[] = {{a.q, a.qs, {a.T, a.m, a.H}},         {a.k, a.ks, {a.T, a.Hkv, a.Lmax}}, {a.v, a.vs, {a.T, a.Hkv, a.Lmax}},
           {a.kd, a.kds, {a.T, a.m, a.Hkv}}, {a.vd, a.vds, {a.T, a.m, a.Hkv}}};
  for (const auto& x : t) {
    if (!aligned(x.p, 16)) return false;
    for (int u = 0; u < 3; ++u)
      if (x.n[u] > 1 && (x.s[u] <= 0 || x.s[u] % 8 != 0 || x.s[u] >= (1ll << 38))) return false;
  }
  return true;
}

// Tensor map of 16-bit elements [n2][n1][n0][d], strides in elements, 64-column boxes.
static bool tree_map(CUtensorMap* map, const void* base, int d, int n0, int64_t s0, int n1, int64_t s1, int n2,
                     int64_t s2, int b0, int b1) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(n0), static_cast<uint64_t>(n1),
                            static_cast<uint64_t>(n2)};
  // the stride of an axis of length 1 is never used, but it is checked
  const uint64_t strides[3] = {n0 > 1 ? s0 * 2ull : 256, n1 > 1 ? s1 * 2ull : 256, n2 > 1 ? s2 * 2ull : 256};
  const uint32_t box[4] = {64, static_cast<uint32_t>(b0), static_cast<uint32_t>(b1), 1};
  return encode_tmap_4d_u16(map, base, dims, strides, box);
}

template <int PANELS, bool BF16>
static int launch_attn_keys(const TreeMmaParams& p, uint32_t smem, cudaStream_t st) {
  const int rc = opt_in<k_tree_attn_keys<PANELS, BF16>>(227 * 1024);
  if (rc != MB_OK) return rc;
  return launch_with_pdl(k_tree_attn_keys<PANELS, BF16>, dim3(p.whole ? p.T * p.a.Hkv * p.RB : p.grid),
                         dim3(kKeysThreads), smem, st, p);
}

template <int PANELS, bool BF16>
static int launch_attn_rows(const TreeMmaParams& p, uint32_t smem, cudaStream_t st) {
  const int rc = opt_in<k_tree_attn_rows<PANELS, BF16>>(227 * 1024);
  if (rc != MB_OK) return rc;
  return launch_with_pdl(k_tree_attn_rows<PANELS, BF16>, dim3(p.whole ? p.T * p.a.Hkv * p.RB : p.grid),
                         dim3(kRowsThreads), smem, st, p);
}

template <int PANELS, bool BF16>
static int launch_rows(const TreeMmaParams& p, uint32_t smem, cudaStream_t st) {
  const int rc = p.n16 == kKeysRows ? launch_attn_keys<PANELS, BF16>(p, smem, st)
                                    : launch_attn_rows<PANELS, BF16>(p, smem, st);
  if (rc != MB_OK || p.whole) return rc;
  const int rows = p.join_passes * kJoinBlock / (PANELS * 16);
  return launch_with_pdl(k_tree_join<PANELS, BF16>, dim3(p.join_by_unit ? p.T * p.a.Hkv * p.RB : p.grid - 1, (p.mb * p.G + rows - 1) / rows), dim3(kJoinBlock),
                         0, st, p);
}

template <int PANELS, bool BF16>
static int launch_weights(const TreeMmaParams& p, uint32_t smem, cudaStream_t st) {
  const int rc = opt_in<k_tree_weights<PANELS, BF16>>(227 * 1024);
  if (rc != MB_OK) return rc;
  return launch_with_pdl(k_tree_weights<PANELS, BF16>, dim3(p.grid), dim3(kWeightThreads), smem, st, p);
}

template <int PANELS, bool BF16>
static int launch_all(const TreeMmaParams& p, uint32_t smem, cudaStream_t st) {
  const int rc = launch_rows<PANELS, BF16>(p, smem, st);
  if (rc != MB_OK || !p.lse) return rc;
  if (p.kept)
    return launch_with_pdl(k_tree_weights_kept,
                           dim3(std::max(1, (p.a.Lmax + 4 * kKeptBlock - 1) / (4 * kKeptBlock)), p.T * p.a.Hkv),
                           dim3(kKeptBlock), 0, st, p);
  return launch_weights<PANELS, BF16>(p, smem, st);
}

int tree_mma_launch(const TreeAttnArgs& a, bool bf16, void* ws, void* stream) {
  TreePlan pl;
  if (!tree_plan(a.T, a.m, a.H, a.Hkv, a.Lmax, a.d, &pl)) return MB_ERR_UNSUPPORTED;
  TreeMmaParams p;
  p.a = a;
  const bool cache = a.Lmax > 0;  // without a cache its maps are never used
  if (!tree_map(&p.mq, a.q, a.d, a.H, a.qs[2], a.m, a.qs[1], a.T, a.qs[0], pl.G, pl.mb) ||
      !tree_map(&p.mkd, a.kd, a.d, a.Hkv, a.kds[2], a.m, a.kds[1], a.T, a.kds[0], 1, a.m) ||
      !tree_map(&p.mvd, a.vd, a.d, a.Hkv, a.vds[2], a.m, a.vds[1], a.T, a.vds[0], 1, a.m) ||
      !tree_map(&p.mk, cache ? a.k : a.kd, a.d, cache ? a.Lmax : 1, a.ks[2], a.Hkv, cache ? a.ks[1] : 128, a.T,
                cache ? a.ks[0] : 128, kTile, 1) ||
      !tree_map(&p.mv, cache ? a.v : a.vd, a.d, cache ? a.Lmax : 1, a.vs[2], a.Hkv, cache ? a.vs[1] : 128, a.T,
                cache ? a.vs[0] : 128, kTile, 1) ||
      !tree_map(&p.mk_end, cache ? a.k : a.kd, a.d, cache ? a.Lmax : 1, a.ks[2], a.Hkv, cache ? a.ks[1] : 128, a.T,
                cache ? a.ks[0] : 128, kBox, 1) ||
      !tree_map(&p.mv_end, cache ? a.v : a.vd, a.d, cache ? a.Lmax : 1, a.vs[2], a.Hkv, cache ? a.vs[1] : 128, a.T,
                cache ? a.vs[0] : 128, kBox, 1))
    return MB_ERR_LAUNCH;
  p.G = pl.G;
  p.RB = pl.RB;
  p.mb = pl.mb;
  // measured: a tile of the keys kernel 1,500 cycles (three quarters at d <= 64), of the rows
  // kernel 2,000 when the constants of share_mode were measured (1,800 since either half of a tile keeps
  // its own reference; the constants stand as they were measured together); 128 keys and values of
  // 128 bytes-a-row panels at 6.4 TB/s, 148 SMs
  p.tile_cycles = pl.n16 > kKeysRows ? 2000 : pl.panels == 2 ? 1500 : 1100;
  p.tile_traffic = pl.panels == 2 ? 2900 : 1450;
  if (pl.RB > 1) p.tile_traffic /= pl.RB;  // the row blocks share their keys' traffic
  p.n16 = pl.n16;
  p.used = pl.used;
  p.grid = pl.grid;
  p.nst = pl.nst;
  p.nq = pl.nq;
  p.vec_out = aligned(a.out, 16) && a.os[0] % 8 == 0 && a.os[1] % 8 == 0 && a.os[2] % 8 == 0;
  char* w = static_cast<char*>(ws);
  p.part = reinterpret_cast<float*>(w);
  w += static_cast<size_t>(2) * pl.grid * pl.mb * pl.G * pl.panels * 64 * 4;
  p.ml = reinterpret_cast<float*>(w);
  w += static_cast<size_t>(2) * pl.grid * 2 * kMaxRows * 4;
  // join CTAs that find a unit to join: about as many as the GPU holds at once
  const int per_pass = kJoinBlock / (pl.panels * 16), groups = (pl.mb * pl.G + per_pass - 1) / per_pass;
  const int64_t cuts = std::min<int64_t>(static_cast<int64_t>(a.T) * a.Hkv * pl.RB, pl.grid - 1);
  p.join_passes = static_cast<int>(std::max<int64_t>(1, cuts * groups / (4 * pl.grid)));
  p.lse = p.kept = p.kept_draft = nullptr;
  p.kept_len = (a.Lmax + 3) / 4 * 4;
  if (a.scores_out) {
    p.lse = reinterpret_cast<float*>(w);
    w += static_cast<size_t>(a.T) * a.Hkv * pl.RB * kMaxRows * 4;
    if (pl.mb * pl.G <= kKeptRows) {  // RB = 1: units are (trace, KV head)
      p.kept_draft = reinterpret_cast<float*>(w);
      p.kept = p.kept_draft + static_cast<size_t>(a.T) * a.Hkv * pl.mb * pl.G * 64;
    }
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int t0 = 0; t0 < a.T; t0 += kMaxTraces) {
    p.t0 = t0;
    p.T = std::min(kMaxTraces, a.T - t0);
    p.whole = a.Lmax <= kWholeRows && p.T * a.Hkv * pl.RB <= pl.grid;
    // Few units have a join CTA each; more units than boundaries, or so few that their CTAs would all
    // lie on the first SMs that come free, one per boundary, most with nothing to join. Measured, by
    // unit / by boundary: 32 units of 128 rows, 16 row groups 35.3 / 38.8 us, 64 units 32.3 / 35.1; but 8
    // units of 32 rows, 4 row groups 88.8 / 87.1.
    const int units = p.T * a.Hkv * pl.RB;
    p.join_by_unit = units < pl.grid && units * groups >= pl.grid / 2;
    int rc;
    if (pl.panels == 2)
      rc = bf16 ? launch_all<2, true>(p, pl.smem, st) : launch_all<2, false>(p, pl.smem, st);
    else
      rc = bf16 ? launch_all<1, true>(p, pl.smem, st) : launch_all<1, false>(p, pl.smem, st);
    if (rc != MB_OK) return rc;
  }
  return MB_OK;
}

}  // namespace mb
