"""B200-native (sm_100a) fused DeepSeek-V3 FP8 block-scale MoE layer.

``kernelforge_b200.kernel`` is a drop-in for the reference operator
``solution/triton/kernel.py::kernel``; the compute runs in ``libkf_moe.so``.
``kernelforge_b200.train`` has the operators of training around a caller's own expert products
(a packed solution carries the layer alone, without them).
"""
from .binding import experts, kernel, route  # noqa: F401
