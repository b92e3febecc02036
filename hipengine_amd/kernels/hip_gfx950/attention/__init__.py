"""Attention half of a decode or prompt step: q / k norm with rotation, the 8-bit paged KV cache, attention over it."""
