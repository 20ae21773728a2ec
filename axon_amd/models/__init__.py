"""Models: a configuration becomes a `DecoderModel` (every architecture here is a decoder made
of registered parts; what differs between architectures is their configuration class)."""
from ..config.base import ModelConfig
from .decoder import CachePlan, DecoderModel


def build_model_description(config: ModelConfig, cache_bits: int = 0) -> DecoderModel:
    """The model as parts and declarations, before any weight or device memory.  `cache_bits`: 4 has every mixer hold its keys and
    values in 4 bits (a ConfigError if one cannot); 0: in the compute dtype."""
    from .. import parts  # noqa: F401  (registers the built-in parts)
    return DecoderModel(config, cache_bits)


__all__ = ["CachePlan", "DecoderModel", "build_model_description"]
