"""paged_attention_prefix operator family."""
