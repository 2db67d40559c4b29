"""B200 (sm_100a) FP8 flash-attention forward behind the operator interface of
weishengying/cutlass_flash_atten_fp8.  See api.py for the operator, paged_kv.py for the
paged fp8 key/value cache and the attention over it, shard.py for
the (batch x head) partition used on multi-GPU boxes, synth.py for the seeded
synthetic workloads of the benchmark."""
from .api import HostRunner, check_status, flash_attention_v2_cutlass, quantize_e4m3  # noqa: F401
from .paged_kv import PagedKVCache, flash_attention_paged_kv, paged_kv_append, paged_kv_read  # noqa: F401
from .shard import shard_range  # noqa: F401

__all__ = ["flash_attention_v2_cutlass", "check_status", "HostRunner", "quantize_e4m3", "PagedKVCache",
           "paged_kv_append", "paged_kv_read", "flash_attention_paged_kv", "shard_range"]
