"""MI355X-native kernels behind the PyTorch-facing API of alexdremov/kernels.

`kernels_amd/streaming_attention` mirrors `src/streaming_attention` of the reference and `kernels_amd/self_attention` its dense forward;
`cross_attention` and `paged_attention` (shared parts in `kv_attention`) stand beside them.  `kernels_amd/csrc` holds the HIP kernels
and their C ABIs.
"""
