"""pypto_amd -- MI355X (gfx950) implementation of the quantized DeepSeek-V3.2 sparse-attention path.

Operators (same names and signatures as the reference examples they replace):

* :func:`sparse_flash_attention_quant_d` / :func:`sparse_flash_attention_quant_p`
* :func:`sparse_attention_antiquant_d` / :func:`sparse_attention_antiquant_p` (packed 656-byte cache rows)
* :func:`lightning_indexer_decode`
* :func:`lightning_indexer_prolog_quant` (the projection stage in front of the indexer)
* :func:`mla_prolog_quant_d` / :func:`mla_prolog_quant_p` (the projection stage in front of the attention)
* :func:`mla_indexer_prolog_quant_d` / :func:`mla_indexer_prolog_quant_p` (both prologs in one call)

What a prompt needs around them, none of it in the reference:

* :func:`rotary_tables`, :func:`rotary_embedding`, :func:`rotary_frequencies` (rotary positions)
* :func:`latent_cache_write` / :func:`latent_cache_write_packed` (quantising the cache as it is written)
* :func:`latent_cache_read` / :func:`latent_cache_read_packed` (reading it back)
* :func:`prompt_attention`, :func:`prompt_window_attention` (attention over whole sequences in the multi-head form)

What a serving step needs, none of it in the reference:

* :func:`cache_pages`, :func:`cache_slots` (block tables, positions and cache rows from lengths)
* :func:`latent_attention` / :func:`latent_attention_packed` (trees of drafted tokens and windows over the cache)

plus :func:`from_torch`, the tensor hand-over of the reference's jit convention.  The computation
runs in hand-written HIP kernels behind a C ABI (``include/pypto_amd_sfa.h``); there is no CPU
fallback.
"""
from .cache_layout_impl import cache_pages, cache_slots  # noqa: F401
from .converter import Tensor, from_torch  # noqa: F401
from .latent_attention_impl import latent_attention, latent_attention_packed  # noqa: F401
from .latent_cache_impl import (latent_cache_read, latent_cache_read_packed, latent_cache_write,  # noqa: F401
                                latent_cache_write_packed)
from .lightning_indexer_quant_impl import LightningIndexerConfigs, lightning_indexer_decode  # noqa: F401
from .lightning_indexer_prolog_quant_impl import (IndexerPrologQuantAttr, IndexerPrologQuantConfigs,  # noqa: F401
                                                  IndexerPrologQuantInput, IndexerPrologQuantOutput,
                                                  lightning_indexer_prolog_quant)
from .mla_indexer_prolog_quant_impl import mla_indexer_prolog_quant_d, mla_indexer_prolog_quant_p  # noqa: F401
from .mla_prolog_quant_impl import (MlaQuantInputs, MlaTileConfig, RopeTileShapeConfig,  # noqa: F401
                                    mla_prolog_quant_d, mla_prolog_quant_p)
from .prompt_attention_impl import prompt_attention, prompt_window_attention  # noqa: F401
from .rotary_position_impl import (RotaryScaling, rotary_embedding, rotary_frequencies, rotary_magnitude,  # noqa: F401
                                   rotary_tables)
from .sparse_attention_antiquant_impl import sparse_attention_antiquant_d, sparse_attention_antiquant_p  # noqa: F401
from .sparse_flash_attention_quant_impl import (SaTileShapeConfig, sparse_flash_attention_quant_d,  # noqa: F401
                                                sparse_flash_attention_quant_p)

__version__ = "0.8.3"
