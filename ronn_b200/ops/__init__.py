"""Python entry points of the hand-written sm_100a kernels."""
from .kernels import *  # noqa: F401,F403
from .kv8 import KV8Cache, kv8_append, kv8_attention, kv8_prefill_attention, kv8_read  # noqa: F401
from .logprobs import TokenLogprobs, token_logprobs  # noqa: F401
