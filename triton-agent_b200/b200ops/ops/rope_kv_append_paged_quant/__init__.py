"""rope_kv_append_paged_quant operator family."""
