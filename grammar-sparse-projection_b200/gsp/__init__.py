"""B200-native grammar-conditioned LM head (drop-in for the reference's ``gsp`` package).

Modules:
  gsp.triton_runtime  -- reference API for bitmask-conditioned logits (CUDA underneath)
  gsp.runtime         -- reference API for id-list projection (constrained_projection)
  gsp.int8_head       -- the head on int8 weights with scales per vocabulary row and request
  gsp.fp8_head       -- the head on e4m3 weights with scales per 128 x 128 block
  gsp.norm           -- the norm before the head, with the residual's addition and 8-bit outputs
  gsp.logprobs        -- log probabilities of given tokens, entropy and alternatives, with their gradient
  gsp.vocab_parallel  -- the head sharded by vocabulary rows over several GPUs
"""
__all__ = ["triton_runtime", "runtime", "int8_head", "fp8_head", "norm", "logprobs", "vocab_parallel"]
