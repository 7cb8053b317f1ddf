"""Speculative decoding: rejection sampling (the reference's memforge_ml.speculative)
and the accepted path of drafted trees."""

from memforge_amd.speculative.rejection_sampler import RejectionSampler
from memforge_amd.speculative.tree import AcceptedPath, accept_tree

__all__ = ["RejectionSampler", "AcceptedPath", "accept_tree"]
