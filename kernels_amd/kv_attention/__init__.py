"""The native part that ``cross_attention`` and ``paged_attention`` share: the dispatcher ops, their GPU implementation
(csrc/kv_torch.cpp, module ``_native``, on the HIP kernels of libkv_attention.so) and the ctypes loader of the C ABI."""
