"""stride_amd: MI355X-native (gfx950) batch-invariant BF16 linear-layer GEMMs for
the stride inference engine, behind the C ABI of include/stride_tc.h.

    stride_amd.tc      the operator surface (tc_qkv, tc_gemm_residual, tc_mlp13,
                       tc_lm_greedy, tc_lm_full) mirroring src/kernels_tc.h
    stride_amd.layout  tile packing / unpacking of weights and activations
    stride_amd.synth   portable seeded synthetic inputs
    stride_amd.harness runners of single operators, window_attention among them
    stride_amd.kv_pool KV pages that sequences share, reserved, forked and compacted on
                       the device (include/stride_serve.h, as the next two)
    stride_amd.logits  penalties, biases, masks and the greedy choice
    stride_amd.serving the engine over those three
    stride_amd.build   builds libstride_tc.so with hipcc for gfx950
"""
__version__ = "0.1.0"
