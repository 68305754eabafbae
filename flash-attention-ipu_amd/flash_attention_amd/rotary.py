"""Norm of query and key heads with the position rotation, forward and backward, in front of this package's attention.

    table = rotary_table(max_positions, head_dim, device="cuda")
    q, k = qk_norm_rope(q, k, q_weight, k_weight, table, positions)
"""

from ._impl.rotary import qk_norm_rope, rotary_table

__all__ = ["qk_norm_rope", "rotary_table"]
