"""B200-native routed-MoE path of the Moonshine Kimi-K3 engine.

``ops``   - the reference's C operator interface (``k3_rocm_*``) on torch tensors
``layer`` - slot table + fused layer (router, dispatch, grouped experts, combine)
``ep``    - expert-parallel layer over torch.distributed
``fp8``   - linear layers and routed experts on E4M3 tables with a scale per block of 128
``balance`` - counts per expert, balance loss and the gradient of the router
``synth`` - seeded synthetic tensors
"""
__version__ = "0.1.0"
