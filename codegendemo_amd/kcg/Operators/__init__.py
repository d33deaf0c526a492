"""Operators of the kcg mirror: matmul (tuned per size), and an 8-bit serving path whose sizes are run-time arguments
(matmul_fp8, quant: rmsnorm_quant and swiglu_quant, moe: moe_layer)."""
