from .mpt import MPTCausalLM, MPTConfig, build_model
from .shared_prefix import SharedPrefix

__all__ = ["MPTCausalLM", "MPTConfig", "SharedPrefix", "build_model"]
