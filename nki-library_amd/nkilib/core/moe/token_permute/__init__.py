"""Tokens into the order of the block table and back, with routing weights and gradients."""

from .token_permute import build_token_slots, combine_tokens, combine_tokens_bwd, permute_tokens, permute_tokens_bwd

__all__ = ["build_token_slots", "permute_tokens", "permute_tokens_bwd", "combine_tokens", "combine_tokens_bwd"]
