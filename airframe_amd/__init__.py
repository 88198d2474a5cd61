"""airframe_amd -- MI355X (gfx950) INT4 KV-cache path: RoPE-fused quantize-on-append, split-K
GQA decode attention and chunked-prefill attention over the INT4 cache, rotary positions, attention
and cache rows of packed prompts, attention behind a shared prefix, behind the C ABI in
include/turboshimmy.h."""
from ._lib import LIB_PATH, TsError, load  # noqa: F401

__all__ = ["LIB_PATH", "TsError", "load", "KVCache", "RopeTable", "attn_prompt", "attn_prompt_workspace", "rope_apply"]


def __getattr__(name):
    if name in ("KVCache", "RopeTable"):
        from . import kv_cache
        return getattr(kv_cache, name)
    if name in ("attn_prompt", "attn_prompt_workspace", "rope_apply"):
        from . import prompt
        return getattr(prompt, name)
    raise AttributeError(name)
