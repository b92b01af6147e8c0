"""Settings of the engine around a model: precision, cache pool, scheduler limits.

The scheduler limits carry the names and meanings of the reference's
`SchedulerConfig` (src/paged/scheduler.rs:37-60): `max_running_requests` caps the
requests that hold cache at once, `max_batch_tokens` caps the new tokens of one
step.  The reference fixes its pool at 256 pages of 16 tokens
(src/backend/candle.rs:158-165); here the pool is sized by the caller.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

WEIGHT_GROUPS = (32, 64, 128)
DTYPE_NAMES = {"bfloat16": "bfloat16", "bf16": "bfloat16", "float32": "float32", "fp32": "float32", "f32": "float32"}


@dataclass
class EngineConfig:
    dtype: str = "bfloat16"
    device: str = "cuda:0"
    page_size: int = 16
    # Size of the pool: either pages for every group, or a token capacity that
    # each group's page count is derived from.
    num_pages: Optional[int] = None
    max_cache_tokens: Optional[int] = None
    max_running_requests: int = 64
    max_batch_tokens: int = 2048
    # A fixed portion size for prompts (None: whatever the budget leaves).
    chunk_size: Optional[int] = None
    # Longest sequence a request may reach; None: max_position_embeddings.
    max_model_len: Optional[int] = None
    # Capture decode-only steps in CUDA graphs.
    cuda_graphs: bool = True
    seed: int = 0
    # 4: the layers' matrices are made four-bit as they are loaded (scale and offset per `weight_group` neighbours of a row), as the
    # reference can do (src/paged/dyn_quant.rs); None: they keep the engine's element type.  `head_bits` says the same of the output
    # head, which the tokens are most sensitive to (a tied head takes a copy of the embedding's table, which stays as it is).
    weight_bits: Optional[int] = None
    weight_group: int = 64
    head_bits: Optional[int] = None

    def __post_init__(self) -> None:
        if self.dtype not in DTYPE_NAMES:
            raise ValueError("dtype %r is not one of %s" % (self.dtype, sorted(set(DTYPE_NAMES))))
        self.dtype = DTYPE_NAMES[self.dtype]
        if self.page_size <= 0:
            raise ValueError("page_size must be positive")
        if self.max_running_requests <= 0:
            raise ValueError("max_running_requests must be positive")
        if self.max_batch_tokens <= 0:
            raise ValueError("max_batch_tokens must be positive")
        if self.chunk_size is not None and self.chunk_size <= 0:
            raise ValueError("chunk_size must be positive")
        for name in ("weight_bits", "head_bits"):
            if getattr(self, name) not in (None, 4):
                raise ValueError("%s is None or 4, not %r" % (name, getattr(self, name)))
        if self.weight_group not in WEIGHT_GROUPS:
            raise ValueError("weight_group %r is not one of %s" % (self.weight_group, WEIGHT_GROUPS))
        if (self.weight_bits or self.head_bits) and self.dtype != "bfloat16":
            raise ValueError("matrices in four bits go with dtype bfloat16, not %s" % self.dtype)
