"""B200-native grammar-conditioned LM head (drop-in for the reference's ``gsp`` package).

Modules:
  gsp.triton_runtime  -- reference API for bitmask-conditioned logits (CUDA underneath)
  gsp.runtime         -- reference API for id-list projection (constrained_projection)
  gsp.int8_head       -- the head on int8 weights with scales per vocabulary row and request
  gsp.logprobs        -- log probabilities of given tokens, entropy and alternatives, with their gradient
  gsp.vocab_parallel  -- the head sharded by vocabulary rows over several GPUs
"""
__all__ = ["triton_runtime", "runtime", "int8_head", "logprobs", "vocab_parallel"]
