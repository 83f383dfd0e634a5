"""Sums of no rows or no tokens, whose tensors have no address, and batches of none: nothing to
add, to choose or to describe.  Without a GPU: batches of none, so nothing is launched."""

from __future__ import annotations

import pytest

from latentserve_amd import _tree
from tests.test_tree_abi import _add, _decode, _select, _st


@pytest.fixture(scope="module")
def lib():
    return _tree.lib()


@pytest.mark.parametrize("over", [dict(sl=0), dict(ns=0), dict(sl=0, ns=0)])
def test_sums_of_nothing_need_no_address(lib, over):
    assert _decode(lib, s=None, b=0, **over) == 0
    assert _add(lib, s=None, b=0, **over) == 0


def test_selection_from_no_tokens_needs_no_address(lib):
    assert _select(lib, s=None, sl=0, b=0, ss=_st(0, 0, 0)) == 0


def test_sums_of_something_do(lib):
    for call in (_decode, _add, _select):
        assert call(lib, s=None, b=0) == 1 and "null" in lib.ls_last_error().decode()


def test_no_trees_need_no_address(lib):
    assert lib.ls_tree_masks(None, None, None, 0, 5, None) == 0
    assert lib.ls_tree_masks(None, None, None, 1, 5, None) == 1
    assert lib.ls_tree_masks(None, None, None, 0, 257, None) == 1
