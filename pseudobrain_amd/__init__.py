"""MI355X-native Gated DeltaNet operator (prefill, its backward, decode) behind the
reference's operator API; see pseudobrain_amd.gated_deltanet. The layer-side
prologue and epilogue around it are in pseudobrain_amd.layer, the windowed
attention that a hybrid layer runs beside it in pseudobrain_amd.attention, its cache
held in 4 bits in pseudobrain_amd.fp4, the cache's pages in pseudobrain_amd.pages, the
norms and rotation of its queries and keys in pseudobrain_amd.rope."""
from .attention import (  # noqa: F401
    paged_cache_write, paged_decode_attention, window_attention, window_attention_bwd, window_attention_fwd,
)
from .fp4 import (  # noqa: F401
    Fp4Cache, fp4_cache, paged_cache_read_fp4, paged_cache_write_fp4, paged_decode_attention_fp4,
)
from .gated_deltanet import (  # noqa: F401
    CHUNK, KERNELS, SEQUENTIAL_MAX, chunk_bwd, chunk_decumulate, chunk_fwd, chunk_fwd_slots, chunk_residuals,
    chunk_slots_, delta_rule_hip, delta_rule_sequential, gated_delta_chunk, gated_delta_chunk_backward,
    gated_delta_chunk_fla, gated_delta_chunk_fla_backward, gated_delta_rule, hip_usable, recurrent_fwd,
    recurrent_step_, register_reference_ops, select_kernel,
)
from .layer import decode_layer_step, layer_epilogue, layer_prologue, layer_prologue_varlen  # noqa: F401,E402
from .pages import paged_cache_extend, paged_cache_release  # noqa: F401,E402
from .rope import qk_norm_rope, rope_tables  # noqa: F401,E402
