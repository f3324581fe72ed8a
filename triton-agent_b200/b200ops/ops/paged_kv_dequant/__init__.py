"""paged_kv_dequant operator family."""
