"""Operators of the kcg mirror: matmul (tuned per size), and an 8-bit serving path whose sizes are run-time arguments
(matmul_fp8, quant: rmsnorm_quant and swiglu_quant, moe: moe_layer).  The 8-bit ones have no gradient: while torch records gradients
they refuse tensors that require one."""
