"""nuvec_amd — MI355X (gfx950) backend for nuvec's quantized-matmul path.

`libnuvec_hip.so` (C ABI in include/nuvec_hip.h) holds the kernels; `ops` mirrors nuvec's
public `quantize`, `dequantize`, `quantized_matmul` and `gather_qmm`, and the row lookup of
nuvec-nn's `QuantizedEmbedding` as `embedding`; `moe_order`, `moe_route` and `weighted_sum` are the glue of
nuvec-lm's mixture-of-experts blocks around the gathered products; `formats` and `checkpoint` turn checkpoint files
into `Quantized` operands in device memory.  `paged` holds what stands between a model's projections and its
attention: rotary positions with one axis or several, norms of heads, a paged, quantized key / value cache, the attention over it and that of
whole prompts over their own keys and values.  `apply_adapters` adds the low-rank adapters of many requests to a shared
projection, `moe_select` chooses experts from a router's logits.
"""
from .ops import (Adapters, GatherQmm, InvalidArgument, Quant, QuantMode, Quantized, Unsupported, apply_adapters, dequantize, embedding,  # noqa: F401
                  gather_qmm, gather_qmm_glu, gather_qmm_grouped, gather_qqmm, glu, moe_order, pair_rows, moe_route, moe_select, qqmm, quantize, quantize_dequantize,
                  quantized_matmul, quantized_matmul_glu, quantized_matmul_kernel, quantized_matmul_route, quantized_matmul_tile, sorted_offsets, weighted_sum)
from .paged import (PagedCache, Rotation, append_paged, head_norm_rope, paged_attention, prompt_attention, read_paged, rope, rotary_axes, rotation_freqs)  # noqa: F401
