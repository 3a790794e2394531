"""The native part that ``cross_attention``, ``paged_attention`` and ``qk_norm_rope`` share: the dispatcher ops, their GPU implementation
(csrc/kv_torch.cpp and kv_rope_torch.cpp, module ``_native``, on the HIP kernels of libkv_attention.so) and the ctypes loader of the C ABI."""
