"""Choosing the next token from a row of logits."""
