"""Device operators: thin kernel wrappers (``kernels``), autograd functions of the
fused GPT path (``fused``), attention, FP8 quantisation, and the memory-bound
operators around a decoder's matrix products: rotary positions (``rotary``), the
residual update with its norms (``residual_norm``) and log probabilities of given
tokens (``logprobs``)."""
