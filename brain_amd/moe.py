"""The int8 mixture-of-experts feed-forward of a decoder layer: router choice, gated experts, weighted sum.

Six calls for any number of tokens and experts (the route is one to three launches),
with no host synchronisation between them, so a decode step can be captured:

    sx, xq       = quant(x)                          ops.quantize_rows[_bf16]
    weights, plan = route(logits)                     ops.moe_route
    h            = silu(x . gate_e) * (x . up_e)      ops.matmul_i8_grouped_glu
    sx, hq       = quant(h)                          ops.quantize_rows[_bf16]
    y            = h . down_e                        ops.matmul_i8_grouped
    out          = sum_j weights_j * y_j (+ add)      ops.moe_combine

The reference runs one gated linear per expert and projection over all tokens
(crates/kernels/wgsl/moe_linear_gated_i8.wgsl:66-69); here each expert multiplies
the rows that were routed to it and nothing else.
"""
import torch

from . import ops


class MoeInt8:
    """gate_up [n_experts, 2 d_ff, d_model / 4] and down [n_experts, d_model, d_ff / 4]
    int32 words (4 codes each; gate rows first), with their scales per row. The
    router's own product is the caller's: it hands in the logits."""

    def __init__(self, gate_up, gate_up_scale, down, down_scale, top_k, score="softmax", renormalize=True, scale=1.0):
        n_experts, two_ff, kg = gate_up.shape
        if down.shape != (n_experts, 4 * kg, two_ff // 8) or two_ff % 8:
            raise ValueError(f"MoeInt8: gate_up {tuple(gate_up.shape)} and down {tuple(down.shape)} do not fit; d_ff and "
                             "d_model are multiples of 4")
        self.gate_up, self.gate_up_scale, self.down, self.down_scale = gate_up, gate_up_scale, down, down_scale
        self.n_experts, self.d_model, self.d_ff = n_experts, 4 * kg, two_ff // 2
        self.top_k, self.score, self.renormalize, self.scale = top_k, score, renormalize, scale

    @classmethod
    def quantize(cls, gate_up, down, top_k, **router):
        """From f32 weights gate_up [n_experts, 2 d_ff, d_model] and down [n_experts, d_model, d_ff] on the GPU."""
        packed = []
        for w in (gate_up, down):
            wq, sw = ops.quantize_weight_device(w.flatten(0, 1))
            packed += [wq.view(*w.shape[:2], -1), sw.view(w.shape[:2])]
        return cls(*packed, top_k, **router)

    def __call__(self, x, logits, mask=None, add=None):
        """x [tokens, d_model] f32 or bf16, logits [tokens, n_experts]; mask, add as
        in ops.moe_route and ops.moe_combine. Returns [tokens, d_model] of x's dtype."""
        if x.dim() != 2 or x.shape[1] != self.d_model or logits.shape != (x.shape[0], self.n_experts):
            raise ValueError(f"MoeInt8: x {tuple(x.shape)} and logits {tuple(logits.shape)}, expected [tokens, {self.d_model}] "
                             f"and [tokens, {self.n_experts}]")
        quantize = ops.quantize_rows_bf16 if x.dtype == torch.bfloat16 else ops.quantize_rows
        sx, xq = quantize(x)
        weights, _, plan = ops.moe_route(logits, self.top_k, self.score, self.renormalize, self.scale, mask)
        h = ops.matmul_i8_grouped_glu(xq, self.gate_up, sx, self.gate_up_scale, plan.offsets, plan.rows, out_dtype=x.dtype)
        # (Places behind the last one are not written and not read: their codes mean nothing.)
        sx, hq = quantize(h)
        y = ops.matmul_i8_grouped(hq, self.down, sx, self.down_scale, plan.offsets, out_dtype=x.dtype)
        return ops.moe_combine(y, weights, plan.slots, add=add)
