"""gguf_hip - the GGUF quantized linear path on MI355X (gfx950): a C-ABI HIP library
(libgqk.so, include/gguf_hip.h) behind the vLLM GGUF plugin's linear-method surface.

    from gguf_hip import GGUFLinearMethod, dequantize, ggml_dequantize
    from gguf_hip import GGUFFile, load_grouped_layers      # GGUF v3 files -> grouped layers
    from gguf_hip import lora_add, qk_norm_rope, paged_attention, copy_pages, PagePool   # a decode step around it
    from gguf_hip import step_tables, add_rms_norm, tree_attention         # a step of several new tokens per sequence
    from gguf_hip import page_bounds, select_pages                         # the pages of a long cache that are worth reading
"""
from .ops import (  # noqa: F401
    GGUF_TYPES, TYPE_NAMES, GroupedLayer, dequantize, dequantize_tiles, drop_cached_layers, fused_mul_mat_gguf,
    fused_mul_mat_gguf_grouped, ggml_dequantize, grouped_layer_from_packed, mul_mat_grouped, pack_layer, plan,
    prepare_grouped_layer,
    quant_shape, repack_tiles, tiles_bytes, type_info, type_planes, unrepack_tiles,
)
from .linear import GGUFLinearMethod  # noqa: F401
from .gguf_file import GGUFFile, GGUFTensor, ggml_type_size, layer_runs, load_grouped_layers  # noqa: F401
from .adapters import lora_add, pack_adapters  # noqa: F401
from .attention import paged_attention, qk_norm_rope, rope_table, tree_attention  # noqa: F401
from .norm import add_rms_norm, add_rms_norm_fp8  # noqa: F401
from .pages import PagePool, copy_pages  # noqa: F401
from .sparse import page_bounds, select_pages  # noqa: F401
from .steps import StepTables, step_tables  # noqa: F401
