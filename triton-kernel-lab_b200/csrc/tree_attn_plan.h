// What the tree attention's first kernel leaves for the second, which joins the
// parts of cut items (tree_attn_sm100.cu).  The test-only self-test library
// compiles this header too.
#pragma once

namespace tk {

// A cut item (b Hkv + h; -1: none), the run of its first part, that part's slot
// there (0 or 1) and the number of parts, one in each run from there on.
struct alignas(16) TreeCut {
  int item, run, slot, parts;
};

// Whether the entry is a cut item.  A CTA that gave up waiting may have left its
// entries as the workspace held them: nothing outside the parts is read and
// nothing outside the output written, whatever stands there.
__host__ __device__ __forceinline__ bool tree_cut_ok(const TreeCut& c, int items, int runs) {
  return c.item >= 0 && c.item < items && c.run >= 0 && c.run < runs && (c.slot == 0 || c.slot == 1) && c.parts >= 1 &&
         c.parts <= runs - c.run;
}

}  // namespace tk
