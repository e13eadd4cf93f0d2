"""MI355X-native (gfx950) Mamba 4 memory read.

A drop-in for the reference's lm/kernels memory-read API
(``selective_gaussian_memory``, ``selective_decode``,
``selective_initial_state``, ``spd_solve``, ``selective_diagnostics``,
``SelectiveState``, ``SelectiveResult``),
implemented by hand-written HIP kernels behind the C ABI in
``include/mamba4_memread.h``, plus the caller's preprocessing and read gating
(``memory_inputs``, ``gated_read``; lm/models/mamba4.py:183-237, 266-273)
and the order head's gated scan (``order_memory_chunked``, ``order_memory``;
lm/models/mamba4.py:46-95).  Beside them, the retention layer's operators
(``linear_attention``, ``linear_attention_step``, ``group_norm``,
``embedding``) and the selective layer's (``selective_scan``,
``selective_scan_step``, ``causal_conv``, ``causal_conv_step``, ``rms_norm``,
``rms_norm_e4m3``).
"""

from mamba4_amd.attention import (  # noqa: F401
    LinearAttentionResult,
    linear_attention,
    linear_attention_step,
    linear_attention_step_,
)
from mamba4_amd.conv import (  # noqa: F401
    CausalConvResult,
    causal_conv,
    causal_conv_step,
    causal_conv_step_,
)
from mamba4_amd.memory import (  # noqa: F401
    MEMORY_SOLVE,
    SOLVERS,
    SelectiveResult,
    SelectiveState,
    selective_decode,
    selective_decode_,
    selective_diagnostics,
    selective_gaussian_memory,
    selective_initial_state,
    spd_solve,
)
from mamba4_amd.mixer import (  # noqa: F401
    MemoryInputs,
    MixerRead,
    gated_read,
    memory_inputs,
    mixer_read,
)
from mamba4_amd.embedding import embedding  # noqa: F401
from mamba4_amd.flashmamba import mamba3_fused  # noqa: F401
from mamba4_amd.norm import (  # noqa: F401
    RmsNormE4M3Result,
    RmsNormResult,
    group_norm,
    rms_norm,
    rms_norm_e4m3,
)
from mamba4_amd.order import order_memory, order_memory_chunked  # noqa: F401
from mamba4_amd.selective import (  # noqa: F401
    SelectiveScanResult,
    selective_scan,
    selective_scan_step,
    selective_scan_step_,
)

__all__ = [
    "CausalConvResult",
    "LinearAttentionResult",
    "MEMORY_SOLVE",
    "MemoryInputs",
    "MixerRead",
    "RmsNormE4M3Result",
    "RmsNormResult",
    "SOLVERS",
    "SelectiveResult",
    "SelectiveScanResult",
    "SelectiveState",
    "causal_conv",
    "causal_conv_step",
    "causal_conv_step_",
    "embedding",
    "linear_attention",
    "linear_attention_step",
    "linear_attention_step_",
    "mamba3_fused",
    "gated_read",
    "group_norm",
    "memory_inputs",
    "mixer_read",
    "order_memory",
    "order_memory_chunked",
    "rms_norm",
    "rms_norm_e4m3",
    "selective_decode",
    "selective_decode_",
    "selective_diagnostics",
    "selective_gaussian_memory",
    "selective_initial_state",
    "selective_scan",
    "selective_scan_step",
    "selective_scan_step_",
    "spd_solve",
]
