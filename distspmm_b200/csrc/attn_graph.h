// attn_graph.h — attention over a pattern's entries by rows, 16-bit operands (attn_graph.cu).
#pragma once
#include "attn.h"

namespace dsp {
enum AttnPass { kForward, kDq, kDkv };
// Whether attn_graph.cu takes a call of the gather form (else attn.cu's kernels do).
bool graph_on_tensor_cores(int dtype, int dim);
// The pass's kernel over the chunks of d (A for forward and dq, A transposed for dk, dv); cut rows are left in slots as by
// attn.cu's kernels.
void graph_pass(AttnPass pass, const DirView &d, const AttnArgs &a, int dtype, cudaStream_t s);
}  // namespace dsp
