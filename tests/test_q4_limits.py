"""Sizes, layouts and states in which 4-bit calls are taken or refused: host logic."""
import pytest
import torch


def test_blocks_of_few_rows_are_chosen_for_as_many_as_a_launch_takes():
    """The few-row kernel's launch counts 65535 blocks of 16 rows: of more, a product goes by the tiles."""
    from estudiocanciones_amd import _ffi
    L = _ffi.lib()
    most = 16 * 65535
    few = False
    for N, K in [(8, 1024), (16, 1024), (16, 8192), (48, 192), (250, 64), (1001, 192)]:
        for choice in (lambda M: L.ecd_mm_q4_choice(M, N, K), lambda M: L.ecd_mm_q4_norm_choice(M, N, K, 0),
                       lambda M: L.ecd_mm_q4_norm_choice(M, N, K, 1)):
            few |= bool(choice(most) & 16)
            for M in (most + 1, 1_100_000, 3_000_000):
                p = choice(M)
                assert p > 0 and not p & 16, (M, N, K, p)
    assert few  # (the rule above is what decides)
