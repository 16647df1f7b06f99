// seq_simt.cu -- K6 over all keys of a sequence, packed or in pages.
#include "seq_simt.cuh"

namespace attnb {

void seq_simt_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  if (a.sel_blocks) seq_simt_blocks_launch(a, ctas, s);
  else simt_launch<false>(a, ctas, s);
}

}  // namespace attnb
