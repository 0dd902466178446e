// attn_tile.h — attention over the tile form of a pattern (attn_tile.cu).
#pragma once
#include "attn.h"

namespace dsp {
// Whether a call takes the tile form: the pattern has one, 16-bit operands, dim 64 or 128, no strides of zero.
bool tile_form(const dsp_pattern *p, const dsp_attn_desc *d);
int64_t tile_forward_bytes(const dsp_pattern *p, const dsp_attn_desc *d);
int tile_forward(const dsp_pattern *p, const AttnArgs &a, int dtype, void *ws, cudaStream_t s);
int64_t tile_grad_bytes(const dsp_pattern *p, const dsp_attn_desc *d);
int tile_gradients(const dsp_pattern *p, const AttnArgs &a, int dtype, void *ws, cudaStream_t s);
}  // namespace dsp
