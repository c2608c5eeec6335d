// Drafted decoding over a KV cache on B200 (sm_100a): attention of a tree of drafted
// tokens, and acceptance of the verified tree with the append of its accepted rows.
//
// One trace t holds lens[t] committed rows in its cache and m drafted tokens (nodes of a
// tree in topological order, node 0 its root) whose keys and values lie in draft buffers.
// Node i sees every committed row and the nodes in its 64-bit mask (its ancestors and
// itself):
//   x_l = scale * q_i . k_l,   p = softmax of x over the visible l,   out_i = sum_l p_l v_l.
// Query heads h = kvh * G + g share the keys of KV head kvh (G = H / Hkv).
// Optionally every row's attention weight, summed over the nodes and the G heads of its
// KV head, is added to the row's running score.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "tree.cuh"

namespace mb {

// ---------------------------------------------------------------------------
// What the tensor-core path (tree_mma.cu) does not take: head dims above 128 or no multiple of
// 8, strides or addresses off 16 bytes, broadcast axes, groups of more than 128 heads. A CTA has
// eight rows (nodes x heads of a group) of a KV head and a span of its keys, with fp32 online
// softmax over chunks of 128; spans are joined by k_tree_any_join. A warp's lanes lie along the
// head dim, four keys at a time, so that any alignment is read in whole lines, and share out the
// sums of 8 x 4 products by halving. Bound by instructions (two bytes per load, fp32 FMAs). Measured:
// 16 traces x 16 heads x 2,048 rows of 256, one node / eight nodes over 4 KV heads 744 / 679 us (a key per
// thread, one row per CTA: 2,630 / 4,850); one trace of 16,000 rows 402 us.
// ---------------------------------------------------------------------------
constexpr int kAnyBlock = 128;
constexpr int kMaxHeadDim = 256;

template <bool BF16>
__device__ __forceinline__ float to_f32(uint16_t x) {
  if (BF16) return __uint_as_float(static_cast<uint32_t>(x) << 16);
  return __half2float(__ushort_as_half(x));
}

template <bool BF16>
__device__ __forceinline__ uint16_t from_f32(float x) {
  if (BF16) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

// Key row l of (t, kvh): committed rows first, then the draft's nodes.
__device__ __forceinline__ const uint16_t* tree_row(const uint16_t* cache, const int64_t* cs, const uint16_t* draft,
                                                    const int64_t* ds, int t, int kvh, int len, int l) {
  if (l < len) return cache + t * cs[0] + kvh * cs[1] + l * cs[2];
  return draft + t * ds[0] + (l - len) * ds[1] + kvh * ds[2];
}

constexpr int kLaneDims = kMaxHeadDim / 32;

// A row's elements lane, lane + 32, ..., 0 beyond the head dim. Loads without a condition: one
// in a branch is waited for before the next starts.
template <bool BF16>
__device__ __forceinline__ void load_lane_row(float* r, const uint16_t* row, int d, int lane) {
  uint16_t x[kLaneDims];
#pragma unroll
  for (int u = 0; u < kLaneDims; ++u) x[u] = row[min(lane + 32 * u, d - 1)];
#pragma unroll
  for (int u = 0; u < kLaneDims; ++u) r[u] = lane + 32 * u < d ? to_f32<BF16>(x[u]) : 0.0f;
}

__device__ __forceinline__ float lane_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The warp's sum of v[lane]: each step hands over half of the values that are left.
__device__ __forceinline__ float lane_sums32(float* v, int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = lane & o ? v[i] : v[i + o], keep = lane & o ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

constexpr int kAnyRows = 8;
struct AnySpans {
  float* part;  // [splits][rows of all units][d] unnormalised outputs, where splits > 1
  float* ml;    // [splits][rows of all units][2] their maxima (log2 units) and sums
  float* lse;   // [t, h, i] log2 units, +inf for a node that sees nothing; or null
  int splits, span, groups;
};

// Output and lse of row r (node x group + head of the group) of a unit.
template <bool BF16>
__device__ __forceinline__ void any_output(const TreeAttnArgs& a, float* lse, int unit, int r, int c, float acc,
                                           float top, float sum) {
  const int G = a.H / a.Hkv, t = unit / a.Hkv, i = r / G, h = (unit % a.Hkv) * G + r % G;
  if (c < a.d)
    a.out[t * a.os[0] + i * a.os[1] + h * a.os[2] + c] = from_f32<BF16>(sum == 0.0f ? 0.0f : acc / sum);
  if (lse && c == 0)
    lse[(static_cast<int64_t>(t) * a.H + h) * a.m + i] = sum == 0.0f ? INFINITY : top + log2f(sum);
}

template <bool BF16>
__global__ void __launch_bounds__(kAnyBlock) k_tree_attn_any(const __grid_constant__ TreeAttnArgs a,
                                                             const __grid_constant__ AnySpans s) {
  __shared__ __align__(16) float p[kAnyBlock * kAnyRows];  // [key][row]
  __shared__ float fade_s[kAnyRows], top_s[kAnyRows], sum_s[kAnyRows];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % s.splits, grp = blockIdx.x / s.splits % s.groups;
  const int unit = blockIdx.x / (s.splits * s.groups), t = unit / a.Hkv, kvh = unit % a.Hkv;
  const int G = a.H / a.Hkv, R = a.m * G, r0 = grp * kAnyRows;
  const int len = max(0, min(a.lens[t], a.Lmax));
  const int begin = split * s.span, end = min(len + a.m, begin + s.span);
  float q[kAnyRows][kLaneDims];
#pragma unroll
  for (int r = 0; r < kAnyRows; ++r) {
    const int row = min(r0 + r, R - 1);
    load_lane_row<BF16>(q[r], a.q + t * a.qs[0] + (row / G) * a.qs[1] + (kvh * G + row % G) * a.qs[2], a.d, lane);
  }
  // after the halving a lane has the score of row lane / 4 for one of the four keys
  const int my_row = r0 + (lane >> 2);
  const uint64_t mask = my_row < R ? a.masks[t * a.mask_stride + my_row / G] : 0;
  float acc[kAnyRows][kMaxHeadDim / kAnyBlock] = {};
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {};  // of rows warp and warp + 4
  for (int l0 = begin; l0 < end; l0 += kAnyBlock) {
#pragma unroll 1
    for (int e = 0; e < 32; e += 4) {
      float k[4][kLaneDims], dot[32];
      const int key = warp * 32 + e;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        load_lane_row<BF16>(k[u], tree_row(a.k, a.ks, a.kd, a.kds, t, kvh, len, min(l0 + key + u, end - 1)), a.d, lane);
#pragma unroll
      for (int r = 0; r < kAnyRows; ++r) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          float x = 0.0f;
#pragma unroll
          for (int v = 0; v < kLaneDims; ++v) x = fmaf(q[r][v], k[u][v], x);
          dot[r * 4 + u] = x;
        }
      }
      const float x = lane_sums32(dot, lane) * a.scale_log2;
      const int at = key + (lane & 3), l = l0 + at;
      const bool seen = mask != 0 && l < end && (l < len || (mask >> (l - len)) & 1);
      p[at * kAnyRows + (lane >> 2)] = seen ? x : -INFINITY;
    }
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int r = warp + 4 * y;
      float x[4], mx = top[y], all = 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] = p[(lane + 32 * u) * kAnyRows + r];
        mx = fmaxf(mx, x[u]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float base = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: every weight is 0
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = exp2f(x[u] - base);
        p[(lane + 32 * u) * kAnyRows + r] = w;
        all += w;
      }
      const float fade = exp2f(top[y] - base);
      sum[y] = sum[y] * fade + lane_sum(all);
      top[y] = mx;
      if (lane == 0) fade_s[r] = fade;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kAnyRows; ++r) {
#pragma unroll
      for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u) acc[r][u] *= fade_s[r];
    }
    const int n = min(kAnyBlock, end - l0);
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += 8) {
      uint16_t v[8][kMaxHeadDim / kAnyBlock];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t* row = tree_row(a.v, a.vs, a.vd, a.vds, t, kvh, len, l0 + min(j0 + e, n - 1));
#pragma unroll
        for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u) v[e][u] = row[min(tid + u * kAnyBlock, a.d - 1)];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float4 w0 = *reinterpret_cast<const float4*>(p + (j0 + e) * kAnyRows);
        const float4 w1 = *reinterpret_cast<const float4*>(p + (j0 + e) * kAnyRows + 4);
        const float w[kAnyRows] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u) {
          const float x = to_f32<BF16>(v[e][u]);
#pragma unroll
          for (int r = 0; r < kAnyRows; ++r)  // what a row without weight holds is not used
            acc[r][u] = fmaf(w[r], w[r] != 0.0f ? x : 0.0f, acc[r][u]);
        }
      }
    }
    __syncthreads();
  }
  if (lane == 0) {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      top_s[warp + 4 * y] = top[y];
      sum_s[warp + 4 * y] = sum[y];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kAnyRows; ++r) {
    if (r0 + r >= R) break;
    const int64_t at = (static_cast<int64_t>(split) * a.T * a.Hkv + unit) * R + r0 + r;
#pragma unroll
    for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u) {
      const int c = tid + u * kAnyBlock;
      if (s.splits == 1)
        any_output<BF16>(a, s.lse, unit, r0 + r, c, acc[r][u], top_s[r], sum_s[r]);
      else if (c < a.d)
        s.part[at * a.d + c] = acc[r][u];
    }
    if (s.splits > 1 && tid < 2) s.ml[at * 2 + tid] = tid ? sum_s[r] : top_s[r];
  }
}

// One CTA per row of a unit: its spans, in order.
template <bool BF16>
__global__ void __launch_bounds__(kAnyBlock) k_tree_any_join(const __grid_constant__ TreeAttnArgs a,
                                                             const __grid_constant__ AnySpans s) {
  pdl_wait();
  pdl_launch_dependents();
  const int R = a.m * (a.H / a.Hkv);
  const int64_t rows = static_cast<int64_t>(a.T) * a.Hkv * R, at = blockIdx.x;
  float top = -INFINITY, sum = 0.0f, acc[kMaxHeadDim / kAnyBlock] = {};
  for (int k = 0; k < s.splits; ++k) top = fmaxf(top, s.ml[(k * rows + at) * 2]);
  for (int k = 0; k < s.splits; ++k) {
    const int64_t piece = k * rows + at;
    const float part = s.ml[piece * 2 + 1];
    if (part == 0.0f) continue;
    const float f = exp2f(s.ml[piece * 2] - top);
    sum += part * f;
#pragma unroll
    for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u) {
      const int c = threadIdx.x + u * kAnyBlock;
      if (c < a.d) acc[u] += s.part[piece * a.d + c] * f;
    }
  }
#pragma unroll
  for (int u = 0; u < kMaxHeadDim / kAnyBlock; ++u)
    any_output<BF16>(a, s.lse, static_cast<int>(at / R), static_cast<int>(at % R), threadIdx.x + u * kAnyBlock, acc[u],
                     top, sum);
}

// Weights of the rows, four per warp at a time: their scores against every query of the KV head
// once more, summed in a fixed order (no atomics: the sums repeat bit for bit).
template <bool BF16>
__global__ void __launch_bounds__(kAnyBlock) k_tree_weights_any(TreeAttnArgs a, const float* __restrict__ lse) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = blockIdx.y % a.Hkv, t = blockIdx.y / a.Hkv;
  const int len = max(0, min(a.lens[t], a.Lmax)), total = len + a.m;
  const int G = a.H / a.Hkv;
  const int64_t unit = static_cast<int64_t>(t) * a.Hkv + kvh;
  const int begin = blockIdx.x * kAnyBlock + warp * 32, end = min(total, begin + 32);
  for (int l0 = begin; l0 < end; l0 += 4) {
    float k[4][kLaneDims], w[4] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u)
      load_lane_row<BF16>(k[u], tree_row(a.k, a.ks, a.kd, a.kds, t, kvh, len, min(l0 + u, end - 1)), a.d, lane);
    for (int i = 0; i < a.m; ++i) {
      const uint64_t mask = a.masks[t * a.mask_stride + i];
      if (mask == 0) continue;
      for (int g = 0; g < G; ++g) {
        const int h = kvh * G + g;
        float q[kLaneDims];
        load_lane_row<BF16>(q, a.q + t * a.qs[0] + i * a.qs[1] + h * a.qs[2], a.d, lane);
        const float norm = lse[(static_cast<int64_t>(t) * a.H + h) * a.m + i];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int l = l0 + u;
          float x = 0.0f;
#pragma unroll
          for (int v = 0; v < kLaneDims; ++v) x = fmaf(q[v] * a.scale_log2, k[u][v], x);
          x = lane_sum(x);
          if (l < len || (l < total && (mask >> (l - len)) & 1)) w[u] += exp2f(x - norm);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int l = l0 + u;
      if (l >= end || lane != u) continue;
      if (l < len)
        a.scores_out[unit * a.Lmax + l] = (a.scores ? a.scores[unit * a.Lmax + l] : 0.0f) + w[u];
      else
        a.draft_scores[unit * a.m + (l - len)] = w[u];
    }
  }
}

// Shares the keys of the general path out: about four CTAs per SM, spans of 256 keys or more.
// Returns the bytes of workspace and, with `spans`, lays them out in `ws`.
static size_t any_plan(int T, int m, int H, int Hkv, int Lmax, int d, void* ws, AnySpans* spans) {
  const int R = m * (H / Hkv), groups = (R + kAnyRows - 1) / kAnyRows;
  const int64_t ctas = static_cast<int64_t>(T) * Hkv * groups, keys = static_cast<int64_t>(Lmax) + m;
  int64_t splits = std::min<int64_t>(4 * sm_count() / ctas, (keys + 255) / 256);
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, 64));
  const int64_t span = ((keys + splits - 1) / splits + kAnyBlock - 1) / kAnyBlock * kAnyBlock;
  splits = (keys + span - 1) / span;
  auto bytes = [](size_t n) { return (n * 4 + 255) / 256 * 256; };
  const size_t rows = static_cast<size_t>(T) * H * m, pieces = splits > 1 ? splits * rows : 0;
  if (spans) {
    char* w = static_cast<char*>(ws);
    *spans = {reinterpret_cast<float*>(w + bytes(rows)), reinterpret_cast<float*>(w + bytes(rows) + bytes(pieces * d)),
              reinterpret_cast<float*>(w), static_cast<int>(splits), static_cast<int>(span), groups};
  }
  return bytes(rows) + bytes(pieces * d) + bytes(pieces * 2);
}

// ---------------------------------------------------------------------------
// Acceptance
// ---------------------------------------------------------------------------
struct AcceptArgs {
  const int32_t *tokens, *parents, *target, *lens, *next_pos;
  uint16_t *k, *v;
  const uint16_t *kd, *vd;
  int64_t ks[4], vs[4], kds[4], vds[4];  // element strides: caches (layer, t, h, l), drafts (layer, t, i, h)
  float* scores;
  const float* draft_scores;
  int32_t* positions;
  int32_t *path, *counts, *next_ids, *lens_out, *pos_out;
  uint32_t* err;
  int64_t parent_stride;
  int layers, T, m, Hkv, Lmax, d, heads_per;
  bool vec;  // 16-byte pieces of rows
};

constexpr int kAcceptBlock = 256;

// The accepted path of trace t, found by one warp: from the root, the first child whose
// drafted token is what the model chose at its parent. Returns the number of nodes.
__device__ __forceinline__ int walk_tree(const AcceptArgs& a, int t, int lane, int* path, int* next_id) {
  const int32_t* tok = a.tokens + static_cast<int64_t>(t) * a.m;
  const int32_t* par = a.parents + t * a.parent_stride;
  const int32_t* tgt = a.target + static_cast<int64_t>(t) * a.m;
  int token[2], parent[2], target[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = lane + 32 * u;
    token[u] = i < a.m ? tok[i] : -1;
    parent[u] = i < a.m ? par[i] : -1;
    target[u] = i < a.m ? tgt[i] : -1;
  }
  if (__shfl_sync(0xffffffffu, token[0], 0) < 0) return 0;  // an idle trace
  int cur = 0, n = 0;
  for (;;) {
    if (lane == 0) path[n] = cur;
    ++n;
    const int want = __shfl_sync(0xffffffffu, cur < 32 ? target[0] : target[1], cur & 31);
    *next_id = want;
    const uint32_t lo = __ballot_sync(0xffffffffu, token[0] >= 0 && lane > cur && parent[0] == cur && token[0] == want);
    const uint32_t hi =
        __ballot_sync(0xffffffffu, token[1] >= 0 && lane + 32 > cur && parent[1] == cur && token[1] == want);
    if (!(lo | hi)) return n;
    cur = lo ? __ffs(lo) - 1 : __ffs(hi) + 31;  // larger than the last one: at most m steps
  }
}

// One CTA per (trace, layer) and group of KV heads: the walk, a chain of dependent steps, is
// repeated per CTA, so a CTA does many heads' rows (24 layers of 16 traces and 16 heads: 9.4 us with
// one CTA per head, 7.4 us so). Latency-bound: tokens, the walk, rows, stores.
__global__ void __launch_bounds__(kAcceptBlock) k_tree_accept(const __grid_constant__ AcceptArgs a) {
  __shared__ int path[64];
  __shared__ int count_s;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x;
  const int t = blockIdx.x, layer = blockIdx.y;
  const int h0 = blockIdx.z * a.heads_per, heads = min(a.heads_per, a.Hkv - h0);
  const int len = a.lens[t], pos = a.next_pos[t];
  if (tid < 32) {
    int next_id = -1;
    int n = walk_tree(a, t, tid, path, &next_id);
    if (len < 0 || n > a.Lmax - len) {  // no room: the trace stays as it is
      n = 0;
      next_id = -1;
      if (tid == 0 && a.err) atomicOr(a.err, MB_DEVERR_INDEX);
    }
    if (tid == 0) count_s = n;
    __syncwarp();
    if (layer == 0 && blockIdx.z == 0) {
      for (int j = tid; j < a.m; j += 32) a.path[static_cast<int64_t>(t) * a.m + j] = j < n ? path[j] : -1;
      if (tid == 0) {
        a.counts[t] = n;
        a.next_ids[t] = next_id;
        a.lens_out[t] = len + n;
        a.pos_out[t] = pos + n;
      }
    }
  }
  __syncthreads();
  const int n = count_s;
  if (n == 0) return;
  const uint16_t* kd = a.kd + layer * a.kds[0] + t * a.kds[1] + h0 * a.kds[3];
  const uint16_t* vd = a.vd + layer * a.vds[0] + t * a.vds[1] + h0 * a.vds[3];
  uint16_t* k = a.k + layer * a.ks[0] + t * a.ks[1] + h0 * a.ks[2] + len * a.ks[3];
  uint16_t* v = a.v + layer * a.vs[0] + t * a.vs[1] + h0 * a.vs[2] + len * a.vs[3];
  if (a.vec) {
    const int per = a.d / 8, total = heads * n * per;
    constexpr int kU = 4;  // pieces of both caches in flight per thread
    for (int e0 = tid; e0 < total; e0 += kU * kAcceptBlock) {
      uint4 x[kU], y[kU];
      int64_t to_k[kU], to_v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int e = e0 + u * kAcceptBlock;
        if (e < total) {
          const int r = e / per, c = (e - r * per) * 8, h = r / n, j = r - h * n;
          x[u] = *reinterpret_cast<const uint4*>(kd + path[j] * a.kds[2] + h * a.kds[3] + c);
          y[u] = *reinterpret_cast<const uint4*>(vd + path[j] * a.vds[2] + h * a.vds[3] + c);
          to_k[u] = h * a.ks[2] + j * a.ks[3] + c;
          to_v[u] = h * a.vs[2] + j * a.vs[3] + c;
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (e0 + u * kAcceptBlock < total) {
          *reinterpret_cast<uint4*>(k + to_k[u]) = x[u];
          *reinterpret_cast<uint4*>(v + to_v[u]) = y[u];
        }
    }
  } else {
    const int64_t total = static_cast<int64_t>(heads) * n * a.d;
    for (int64_t e = tid; e < total; e += kAcceptBlock) {
      const int r = static_cast<int>(e / a.d), c = static_cast<int>(e - static_cast<int64_t>(r) * a.d);
      const int h = r / n, j = r - h * n;
      k[h * a.ks[2] + j * a.ks[3] + c] = kd[path[j] * a.kds[2] + h * a.kds[3] + c];
      v[h * a.vs[2] + j * a.vs[3] + c] = vd[path[j] * a.vds[2] + h * a.vds[3] + c];
    }
  }
  const int64_t unit0 = (static_cast<int64_t>(layer) * a.T + t) * a.Hkv + h0;
  for (int e = tid; e < heads * n; e += kAcceptBlock) {
    const int h = e / n, j = e - h * n;
    const int64_t row = (unit0 + h) * a.Lmax + len + j;
    if (a.scores) a.scores[row] = a.draft_scores[(unit0 + h) * a.m + path[j]];
    if (a.positions) a.positions[row] = pos + j;
  }
}

// RoPE of a drafted tree's queries and keys at next_pos[t] + depth[i]: adjacent pairs, as
// mb_rope_append. One CTA per (head of q and k, node, trace).
template <bool BF16>
__global__ void __launch_bounds__(64) k_tree_rope(const uint16_t* __restrict__ qkv, int m, int H, int Hkv, int dh,
                                                  const int32_t* __restrict__ next_pos,
                                                  const int32_t* __restrict__ depth, int64_t depth_stride,
                                                  const float2* __restrict__ cs, int positions,
                                                  uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_out,
                                                  uint32_t* err) {
  pdl_wait();
  pdl_launch_dependents();
  const int h = blockIdx.x, i = blockIdx.y, t = blockIdx.z;
  const int64_t row = static_cast<int64_t>(t) * m + i;
  const int p = next_pos[t] + depth[t * depth_stride + i];
  const uint16_t* src = qkv + row * (H + 2 * Hkv) * dh + h * dh;
  uint16_t* dst = h < H ? q_out + (row * H + h) * dh : k_out + (row * Hkv + (h - H)) * dh;
  if (p < 0 || p >= positions) {
    if (threadIdx.x == 0 && err) atomicOr(err, MB_DEVERR_INDEX);
    return;
  }
  for (int c = threadIdx.x; c < dh / 2; c += 64) {
    const float2 r = cs[static_cast<int64_t>(p) * (dh / 2) + c];
    const float x = to_f32<BF16>(src[2 * c]), y = to_f32<BF16>(src[2 * c + 1]);
    dst[2 * c] = from_f32<BF16>(x * r.x - y * r.y);
    dst[2 * c + 1] = from_f32<BF16>(x * r.y + y * r.x);
  }
}

}  // namespace mb

using namespace mb;

extern "C" {

size_t mb_tree_attn_workspace_size(int32_t T, int32_t m, int32_t H, int32_t Hkv, int32_t Lmax, int32_t d,
                                   int32_t with_scores) {
  if (T < 1 || m < 1 || m > 64 || Hkv < 1 || H < Hkv || H % Hkv != 0 || Lmax < 0 || d < 1 || d > kMaxHeadDim) return 0;
  return std::max(any_plan(T, m, H, Hkv, Lmax, d, nullptr, nullptr), tree_mma_workspace(T, m, H, Hkv, Lmax, d, with_scores != 0));
}

int32_t mb_tree_attn(const mb_tree_attn_args* g, void* stream) {
  if (!g || !g->q || !g->lens || !g->k_draft || !g->v_draft || !g->masks || !g->out) return MB_ERR_NULL;
  const int T = g->T, m = g->m, H = g->H, Hkv = g->Hkv, Lmax = g->Lmax, d = g->d;
  if (Lmax > 0 && (!g->k_cache || !g->v_cache)) return MB_ERR_NULL;
  const bool weights = g->draft_scores != nullptr;  // without a cache there are no other scores
  if ((g->scores_out != nullptr) != weights && !(weights && Lmax == 0)) return MB_ERR_NULL;
  if (g->scores && !g->scores_out) return MB_ERR_NULL;
  if (T < 1 || m < 1 || m > 64 || Hkv < 1 || H < Hkv || H % Hkv != 0 || Lmax < 0 || d < 1 || d > kMaxHeadDim)
    return MB_ERR_ARGS;
  if (static_cast<int64_t>(T) * m * H > 0x7FFFFFFFll || static_cast<int64_t>(T) * Hkv > 65535 || Lmax > 0x7FFF0000)
    return MB_ERR_UNSUPPORTED;
  if (broadcast(g->strides + 15, {T, m, H})) return MB_ERR_ARGS;
  if (weights && g->out == g->q) return MB_ERR_ARGS;  // the weights read q after the outputs are there
  if (!(g->scale - g->scale == 0.0f) || g->is_bf16 < 0 || g->is_bf16 > 1) return MB_ERR_ARGS;
  if (!aligned(g->q, 2) || !aligned(g->k_cache, 2) || !aligned(g->v_cache, 2) || !aligned(g->k_draft, 2) ||
      !aligned(g->v_draft, 2) || !aligned(g->out, 2) || !aligned(g->lens, 4) || !aligned(g->masks, 8) ||
      !aligned(g->scores, 4) || !aligned(g->scores_out, 4) || !aligned(g->draft_scores, 4) || !aligned(g->dev_err, 4))
    return MB_ERR_ALIGN;
  if (!g->workspace ||
      g->workspace_bytes < mb_tree_attn_workspace_size(T, m, H, Hkv, Lmax, d, weights))
    return MB_ERR_WORKSPACE;
  if (!aligned(g->workspace, 16)) return MB_ERR_ALIGN;
  TreeAttnArgs a;
  a.q = g->q;
  a.k = g->k_cache;
  a.v = g->v_cache;
  a.kd = g->k_draft;
  a.vd = g->v_draft;
  a.out = g->out;
  a.lens = g->lens;
  a.masks = reinterpret_cast<const uint64_t*>(g->masks);
  a.mask_stride = g->shared_masks ? 0 : m;
  for (int u = 0; u < 3; ++u) {
    a.qs[u] = g->strides[u];
    a.ks[u] = g->strides[3 + u];
    a.vs[u] = g->strides[6 + u];
    a.kds[u] = g->strides[9 + u];
    a.vds[u] = g->strides[12 + u];
    a.os[u] = g->strides[15 + u];
  }
  a.T = T;
  a.m = m;
  a.H = H;
  a.Hkv = Hkv;
  a.Lmax = Lmax;
  a.d = d;
  a.scale_log2 = g->scale * 1.4426950408889634f;
  a.scores = g->scores;
  a.scores_out = weights && !g->scores_out ? g->draft_scores : g->scores_out;  // Lmax = 0: no row is written
  a.draft_scores = g->draft_scores;
  a.err = g->dev_err;
  const bool bf16 = g->is_bf16 != 0;
  if (tree_mma_workspace(T, m, H, Hkv, Lmax, d, false) && tree_mma_takes(a))
    return tree_mma_launch(a, bf16, g->workspace, stream);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  AnySpans sp;
  any_plan(T, m, H, Hkv, Lmax, d, g->workspace, &sp);
  const int64_t rows = static_cast<int64_t>(T) * H * m;
  const float* lse = sp.lse;
  if (!a.scores_out) sp.lse = nullptr;
  const int64_t ctas = static_cast<int64_t>(T) * Hkv * sp.groups * sp.splits;
  if (ctas > 0x7FFFFFFFll) return MB_ERR_UNSUPPORTED;
  int rc = launch_with_pdl(bf16 ? k_tree_attn_any<true> : k_tree_attn_any<false>, dim3(static_cast<unsigned>(ctas)),
                           dim3(kAnyBlock), 0, st, a, sp);
  if (rc == MB_OK && sp.splits > 1)
    rc = launch_with_pdl(bf16 ? k_tree_any_join<true> : k_tree_any_join<false>, dim3(static_cast<unsigned>(rows)),
                         dim3(kAnyBlock), 0, st, a, sp);
  if (rc != MB_OK || !a.scores_out) return rc;
  return launch_with_pdl(bf16 ? k_tree_weights_any<true> : k_tree_weights_any<false>,
                         dim3((Lmax + m + kAnyBlock - 1) / kAnyBlock, T * Hkv), dim3(kAnyBlock), 0, st, a, lse);
}

int32_t mb_tree_accept(const mb_tree_accept_args* g, void* stream) {
  if (!g || !g->tokens || !g->parents || !g->target || !g->lens || !g->next_pos || !g->k_cache || !g->v_cache ||
      !g->k_draft || !g->v_draft || !g->path || !g->counts || !g->next_ids || !g->lens_out || !g->pos_out)
    return MB_ERR_NULL;
  if ((g->scores != nullptr) != (g->draft_scores != nullptr)) return MB_ERR_NULL;
  const int layers = g->layers, T = g->T, m = g->m, Hkv = g->Hkv, d = g->d;
  if (layers < 1 || T < 1 || m < 1 || m > 64 || Hkv < 1 || g->Lmax < 1 || d < 1) return MB_ERR_ARGS;
  if (g->lens_out == g->lens || g->pos_out == g->next_pos) return MB_ERR_ARGS;  // every CTA reads the old lengths
  for (const int64_t* s : {g->strides, g->strides + 4})
    if ((layers > 1 && s[0] == 0) || broadcast(s + 1, {T, Hkv, g->Lmax})) return MB_ERR_ARGS;
  if (static_cast<int64_t>(T) * layers > 0x7FFFFFFFll || layers > 65535 || Hkv > 65535) return MB_ERR_UNSUPPORTED;
  if (!aligned(g->dev_err, 4)) return MB_ERR_ALIGN;
  AcceptArgs a;
  a.tokens = g->tokens;
  a.parents = g->parents;
  a.parent_stride = g->shared_parents ? 0 : m;
  a.target = g->target;
  a.lens = g->lens;
  a.next_pos = g->next_pos;
  a.k = g->k_cache;
  a.v = g->v_cache;
  a.kd = g->k_draft;
  a.vd = g->v_draft;
  bool vec = d % 8 == 0 && aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.kd, 16) && aligned(a.vd, 16);
  for (int u = 0; u < 4; ++u) {
    a.ks[u] = g->strides[u];
    a.vs[u] = g->strides[4 + u];
    a.kds[u] = g->strides[8 + u];
    a.vds[u] = g->strides[12 + u];
  }
  for (int u = 0; u < 16; ++u) vec = vec && g->strides[u] % 8 == 0;
  a.vec = vec;
  a.scores = g->scores;
  a.draft_scores = g->draft_scores;
  a.positions = g->positions;
  a.path = g->path;
  a.counts = g->counts;
  a.next_ids = g->next_ids;
  a.lens_out = g->lens_out;
  a.pos_out = g->pos_out;
  a.err = g->dev_err;
  a.layers = layers;
  a.T = T;
  a.m = m;
  a.Hkv = Hkv;
  a.Lmax = g->Lmax;
  a.d = d;
  // about two CTAs per SM
  const int groups = std::max(1, std::min<int>(Hkv, 2 * sm_count() / std::max(1, T * layers)));
  a.heads_per = (Hkv + groups - 1) / groups;
  return launch_with_pdl(k_tree_accept, dim3(T, layers, (Hkv + a.heads_per - 1) / a.heads_per), dim3(kAcceptBlock), 0,
                         static_cast<cudaStream_t>(stream), a);
}

int32_t mb_tree_rope(const uint16_t* qkv, int32_t is_bf16, int32_t T, int32_t m, int32_t H, int32_t Hkv, int32_t dh,
                     const int32_t* next_pos, const int32_t* depths, int32_t shared_depths, const float* cs,
                     int32_t positions, uint16_t* q_out, uint16_t* k_out, uint32_t* dev_err, void* stream) {
  if (!qkv || !next_pos || !depths || !cs || !q_out || !k_out) return MB_ERR_NULL;
  if (T < 1 || m < 1 || m > 64 || H < 1 || Hkv < 1 || dh < 2 || dh % 2 != 0 || positions < 1) return MB_ERR_ARGS;
  if (is_bf16 < 0 || is_bf16 > 1) return MB_ERR_ARGS;
  if (T > 65535) return MB_ERR_UNSUPPORTED;
  if (!aligned(cs, 8) || !aligned(dev_err, 4)) return MB_ERR_ALIGN;
  return launch_with_pdl(is_bf16 ? k_tree_rope<true> : k_tree_rope<false>, dim3(H + Hkv, m, T), dim3(64), 0,
                         static_cast<cudaStream_t>(stream), qkv, m, H, Hkv, dh, next_pos, depths,
                         static_cast<int64_t>(shared_depths ? 0 : m), reinterpret_cast<const float2*>(cs), positions,
                         q_out, k_out, dev_err);
}

}  // extern "C"
