// Attention over the 4-bit cache's pages with a view of it: the newest tokens as a tree, of which a
// token sees its ancestors, and windows whose first tokens stay visible.
//
// The formula, the tiles and the split of the work are those of skv_fp4_attention.hip; what
// differs is which positions a row sees.  A token's history is the positions before the new
// ones, then the new ones of its mask (without a tree: those up to itself); it sees the history's
// last `window` and first `first` positions.  Of a row that is a few numbers, worked out once: the
// end hi of what it sees of the old positions, the begin lo of its window, the end `keep` of its
// first tokens (both as positions, found in the mask where they fall among the new ones).  A
// tile is then masked by a word of 32 bits for a row,
//   (below hi, or of the mask) and (not below lo, or below keep),
// and only the tiles at these borders are: the old positions between them are seen by all rows.
// A span's tiles are the first tokens' and the window's, numbered through, so that the ones
// between are neither read nor dealt to a workgroup.  A row whose mask is empty is as the others
// in the tiles that all see, and cleared at the end.
//
// Measured, us a call in a graph of several, with the time of the bytes at 6.1 TB/s or of the products at 1.4 PFLOP/s:
//   trees of up to 32 nodes of 32 sequences of 1k - 16k, 64 heads on 8 of 128 dims   204 (99, products)
//   trees of up to 7 nodes of 4 of 256k - 1M, 16 heads on 4 of 64                    147 (143 - 153; 88)
//   trees of up to 99 nodes of 6, windows of 128, 16 heads on 1 of 512               46 (3, products)
//   64 windows of 4k behind 4 first tokens, 64 heads on 8 of 128                     50 - 56 (44)
//   2 prompts' 1000 tokens, windows of 2k behind 64, 32 heads on 8 of 128            90 (49, products)
//   a tree of 8 nodes over 341 tokens, one token in a window of 128                  9.5, 7.9
#include "skv_fp4_attn.h"

namespace skv {

// Whether v adds nothing to the plain call: without a tree, where no window hides the first tokens.  It is that call then,
// to the bit and in its precision.
inline bool fp4_plain(const skv_fp4_attention_desc* d, const skv_fp4_view* v) {
  return d && !v->tree && (d->window == 0 || v->first == 0);
}

}  // namespace skv

using namespace skv;

extern "C" int64_t skv_fp4_attention_view_workspace(const skv_fp4_attention_desc* d, const skv_fp4_view* v) {
  if (!v) return set_error(SKV_EINVAL, "skv_fp4_attention_view: NULL view"), -1;
  if (fp4_plain(d, v)) return fp4_check_view(d, v) == SKV_OK ? skv_fp4_attention_workspace(d) : -1;
  Fp4AttnPlan p;
  return fp4_attn_plan(d, v, p) == SKV_OK ? p.ws_bytes : -1;
}

extern "C" int skv_fp4_attention_view(const skv_fp4_attention_desc* d, const skv_fp4_view* v, void* workspace, int64_t ws_bytes,
                                      void* stream) {
  if (!v) return set_error(SKV_EINVAL, "skv_fp4_attention_view: NULL view");
  if (fp4_plain(d, v)) {
    const int rc = fp4_check_view(d, v);
    return rc ? rc : skv_fp4_attention(d, workspace, ws_bytes, stream);
  }
  return fp4_attn_call<true>(d, v, workspace, ws_bytes, stream);
}
