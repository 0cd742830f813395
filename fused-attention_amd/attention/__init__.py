"""MI355X (gfx950) fused causal attention with the Python API of the cuTile reference.

attention.fused.fused.fused_attention            causal MHA forward
attention.gqa.fused_gqa.fused_gqa_attention      causal GQA/MQA forward
attention.backward.fused_backward.fused_attention_autograd   forward + recompute backward
attention.rotary.fused_rotary.fused_qk_norm_rotary(_autograd)   norm of q and k with the rotation, and its backward
attention.paged.fused_paged.append_paged_kv, fused_paged_attention   8-bit paged cache and attention over it

All call hand-written HIP kernels in libfa.so, through ctypes or the torch module beside it (attention._lib).
"""
