"""The embedding's C entries of a single table, whose struct says nothing about places (CPU only: no kernel is launched
here)."""

from __future__ import annotations

import ctypes

import pytest

from tests.test_train_abi import _lib, embedding  # noqa: F401  (a fixture)


@pytest.mark.parametrize("period", [0, -1, 1, 7])
def test_no_second_table_takes_no_memory(lib, period):
    """Sizes from which tiles are made, of many tokens and of a large table: without a second table its period, which is
    not read, may be anything, and asking for its gradient adds nothing."""
    for sizes in ({"tokens": 5000}, {"tokens": 40, "vocab": 1 << 24, "dim": 64}, {"tokens": 1 << 30}, {"tokens": 6}, {"tokens": 0}):
        for place_ids in (None, 4096):
            e = dict(sizes, places=0, period=period, place_ids=place_ids)
            for call in (lib.isa_train_embedding_lists, lib.isa_train_embedding_backward_workspace):
                assert call(embedding(**e), 0, 1) == 0
                assert call(embedding(**e), 1, 1) == call(embedding(**e), 1, 0)


def test_gradients_of_a_second_table_that_is_not_there(lib):
    """Past all checks: nothing is left to do, also where tiles would be made."""
    fake = ctypes.c_void_p(4096)
    for tokens in (5000, 1 << 20):
        e = embedding(tokens=tokens, vocab=0)
        size = lib.isa_train_embedding_lists(e, 1, 1)
        ws = lib.isa_train_embedding_backward_workspace(e, 1, 1)
        assert lib.isa_train_embedding_backward(e, fake, size, fake, fake, fake, 1, 1, fake, ws, None) == 0
