// seq_simt_blocks.cu -- K6 over the blocks in a token's list.
#include "seq_simt.cuh"

namespace attnb {

void seq_simt_blocks_launch(const SeqAttnArgs& a, int ctas, cudaStream_t s) {
  simt_launch<true>(a, ctas, s);
}

}  // namespace attnb
