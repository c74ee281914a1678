"""MI355X (gfx950) decode hot path of llmtoy-zig: GGUF block-quantised matvec
and the MoE layer, behind the C ABI in include/llmtoy_hip.h."""
from . import ggml, gguf, synth  # noqa: F401
from .lib import (ACT_GELU_TANH, ACT_SILU, KV_BLOCK, KV_NONE, ROPE_NEOX, ROPE_PAIRS, Context, KvBatch,  # noqa: F401
                  KvCache, LtError, Rope, Tensor, UnsupportedError, load_library, upload_moe)
