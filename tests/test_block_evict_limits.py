"""Evictions that no grid takes are refused before the first of their two launches (no GPU needed: nothing is launched)."""
from inference_engine_rust_b200.csrc import bindings as B


def status(layers, n, kv_heads, keep):
    none = None
    return B.core().iert_block_evict(none, none, none, none, none, layers, 8, kv_heads, 64, 128, none, 4, n, none, none, n, none, -(-keep // 4) + 1, keep, 0,
                                     16, none, none, none, None)


def test_more_blocks_to_copy_than_a_grid_has():
    assert status(65_535, 65_535, 1, 1) == 1          # 2^32 sequences of all layers
    assert status(1_000, 1_000, 8, 4_096) == 1        # 2^22 of them, 513 blocks of threads each
