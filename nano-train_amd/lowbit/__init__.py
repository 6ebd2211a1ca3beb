"""MI355X-native low-bit linear hot path of nano-train (gfx950 HIP kernels behind a C-ABI).

Public surface:
  lowbit.backend.HipLowBitBackend   - the LowBitBackend drop-in ("hip")
  lowbit.ops                        - tensor-level kernel wrappers
  lowbit.contracts                  - the reference's precision value types
  lowbit.norm, .router, .loss       - the high-precision operators around the low-bit products
  lowbit.blocks                     - an MoE block and a small language model of all of them
"""

__all__ = ["backend", "blocks", "contracts", "loss", "norm", "ops", "router"]
