"""Custom flash attention operators (gfx950). Mirrors the reference package
``easyvolcap/utils/custom_flash_attn``; its operators live in ``sparse_index_flash_attn``.
Beside them: ``packed_flash_attn`` (sequences of different lengths, forward and backward) and ``paged_flash_attn``
(new tokens over a paged key-value cache)."""
