"""paged_attention_quant operator family."""
