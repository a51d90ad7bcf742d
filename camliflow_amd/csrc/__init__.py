"""Operator boundary -- the four names the reference exports from ``models/csrc/__init__.py:1``, and the operators of attentive
fusion (cross attention, its bucketed position bias, channels-last group norm), which the reference does not have."""
from .wrapper import correlation2d, furthest_point_sampling, squared_distance, k_nearest_neighbor
from .attention import cross_attention, relative_position_bias
from .norm import group_norm_act

__all__ = ["correlation2d", "furthest_point_sampling", "squared_distance", "k_nearest_neighbor",
           "cross_attention", "relative_position_bias", "group_norm_act"]
