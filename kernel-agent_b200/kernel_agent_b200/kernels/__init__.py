"""The GPU drop-ins of ``kernel_agent.kernels.{quant,compare,scale_guard}`` and the new
blockwise-FP8, FP8-attention, weight-only FP4 and paged FP8 cache APIs."""
