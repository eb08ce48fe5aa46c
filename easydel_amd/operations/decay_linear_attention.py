"""``ragged_decay_linear_attention``: linear attention with one decay per KV head over a ragged batch.

The linear layers of a hybrid decoder, next to its paged attention layers: the same flattened tokens, the same
``query_start_loc`` / ``context_lens`` (``DecayStateMetadata.from_ragged``), and a pool of float32 states in the place of pages.
Prompt chunks, decode rows and mixes of both are one call (``kernels.decay_linear_attention``).
"""

from __future__ import annotations

from .. import kernels
from ..caching.decay_state import DecayStateCacheView, DecayStateMetadata
from ._attention_outputs import AttentionOutput
from ._base_operation import OperationImpl, OperationRegistry
from .requirements import CacheType, ExecutionMode, MetadataField, OperationRequirements, RequirementsBuilder
from .rotary import token_rows


@OperationRegistry.register
class DecayLinearAttn(OperationImpl):
    @classmethod
    def get_impl_name(cls) -> str | tuple[str]:
        return "ragged_decay_linear_attention"

    @classmethod
    def get_requirements(cls, mode: ExecutionMode = ExecutionMode.MIXED) -> OperationRequirements:
        return (RequirementsBuilder("ragged_decay_linear_attention")
                .require_metadata(MetadataField.SEQ_LENS | MetadataField.CONTEXT_LENS | MetadataField.QUERY_START_LOC | MetadataField.STATE_INDICES)
                .support_cache(CacheType.RECURRENT)
                .use_cache_view(DecayStateCacheView)
                .build())

    def forward_native(self, query, key, value, cache_view: DecayStateCacheView, cache_metadata: DecayStateMetadata, log_decay,
                       scale: float | None = None, **ignore) -> AttentionOutput:
        out, state = kernels.decay_linear_attention(
            token_rows(query), token_rows(key), token_rows(value), log_decay, cache_view.state, cache_metadata.state_indices, cache_metadata.query_start_loc,
            cache_metadata.num_seqs, context_lens=cache_metadata.context_lens, state_out_indices=cache_metadata.state_out_indices, scale=scale)
        cache_view.state = state
        return AttentionOutput(attention_weights=None, attention_outputs=out, cache_view=cache_view)

    def __call__(self, query, key, value, cache_view, cache_metadata, log_decay, scale: float | None = None, **ignore) -> AttentionOutput:
        """``query [T, Hq, Dk]`` (or ``[batch, seq, Hq, Dk]``), ``key [T, Hkv, Dk]``, ``value [T, Hkv, Dv]``, ``log_decay [Hkv]`` float32;
        the result has the query's leading shape and ``Dv``-wide heads.  Rows of one projection are read in place, parts of its heads copied."""
        lead = tuple(query.shape[:-1])
        flat = lambda x: x.reshape(-1, *x.shape[-2:]) if x.ndim == 4 else x  # noqa: E731
        output = super().__call__(query=flat(query), key=flat(key), value=flat(value), cache_view=cache_view, cache_metadata=cache_metadata,
                                  log_decay=log_decay, scale=scale, **ignore)
        if query.ndim == 4:
            output.attention_outputs = output.attention_outputs.reshape(*lead, value.shape[-1])
        return output
