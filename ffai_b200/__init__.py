"""ffai_b200: B200-native Whisper attention (encoder self-attention, decoder
self-attention over the KV cache, decoder cross-attention) behind the C ABI
of libffai_attn.so.  See include/ffai_attn.h for the boundary.

    from ffai_b200 import attention, flash_attn
    out = attention.prefill(q, k, v, scale=0.125)          # tcgen05 kernel
    o = attention.decode(q, kcache, vcache, kv_len=448)    # split-KV decode
    o = flash_attn.attend_merged(q, kt, v)                 # reference surface

A batched decode step on the device, from page tables to tokens:

    plan = kvcache.plan_pages(lens, new, free_pages, free_count, table, slot_cap=n)
    kvcache.write_slots(k_pool, v_pool, k_new, v_new, plan.slots)
    o = shared_prefix.attend(q, k_pool, v_pool, prefix_table, prefix_lens, group_starts,
                             table, plan.lens)             # shared prompts read once
    tokens = sampling.sample(logits, u, temperature=t, top_k=k, top_p=p, min_p=m)
    lens, free_count = kvcache.release_pages(plan.lens, done, table, free_pages,
                                             plan.free_count)

group_decoder.GroupDecoder chains them around one attention layer.
"""

from . import _abi  # noqa: F401

__all__ = ["attention", "flash_attn", "partition", "load"]


def load():
    """Load libffai_attn.so (raises ImportError if it has not been built)."""
    return _abi.load()
