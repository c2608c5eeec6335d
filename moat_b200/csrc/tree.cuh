// Arguments and host entry points of the tree attention kernels (tree.cu, tree_mma.cu).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace mb {

struct TreeAttnArgs {
  const uint16_t *q, *k, *v, *kd, *vd;
  uint16_t* out;
  const int32_t* lens;
  const uint64_t* masks;
  int64_t mask_stride;
  // element strides: q / out / drafts (trace, node, head), caches (trace, head, row)
  int64_t qs[3], ks[3], vs[3], kds[3], vds[3], os[3];
  int T, m, H, Hkv, Lmax, d;
  float scale_log2;  // scale * log2(e)
  const float* scores;  // [T, Hkv, Lmax] or null
  float* scores_out;    // [T, Hkv, Lmax] or null
  float* draft_scores;  // [T, Hkv, m] or null
  uint32_t* err;        // optional device error word
};

// Tensor-core path. 0 bytes: the sizes are not among those it takes.
size_t tree_mma_workspace(int T, int m, int H, int Hkv, int Lmax, int d, bool with_scores);
// Whether pointers and strides suit its tensor maps.
bool tree_mma_takes(const TreeAttnArgs& a);
int tree_mma_launch(const TreeAttnArgs& a, bool bf16, void* ws, void* stream);

}  // namespace mb
