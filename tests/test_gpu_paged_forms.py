"""Attention over a paged cache: every number of rows at which another form takes over, with enough
sequences that each form runs, for lengths that differ and for equal ones."""
import pytest
import torch

from . import paged_helpers as P
from .test_gpu_paged_attention import KINDS, _check

pytestmark = pytest.mark.gpu
# rows = q_seq * group on both sides of 16, 32, 64 and 128
ROWS = [(5, 3), (4, 4), (17, 1), (31, 1), (8, 4), (11, 3), (21, 3), (16, 4), (13, 5), (43, 3)]


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", ROWS)
def test_many_units(dtype, packed, head, q_seq, group):
    """36 (sequence, head) pairs, lengths from nothing to some steps; more queries than rows among them."""
    lens = [0, 1, 15, 64, 129, 200, 333, 48, 260]
    _check(P.Case(40, dtype, packed, 9, 4, head, 16, lens, spread=group % 2), q_seq, group)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("q_seq,group", ROWS)
def test_few_units(dtype, packed, q_seq, group):
    """One and two sequences: a unit's keys lie with many workgroups."""
    _check(P.Case(41, dtype, packed, 1, 1, 128, 64, [1777]), q_seq, group)
    _check(P.Case(42, dtype, packed, 2, 2, 64, 32, [900, 411]), q_seq, group, causal=False)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("q_seq,group", [(1, 1), (2, 9), (5, 8), (16, 4)])
@pytest.mark.parametrize("length", [64, 257, 300])
def test_equal_lengths(dtype, packed, head, q_seq, group, length):
    _check(P.Case(43, dtype, packed, 9, 4, head, 64, [length] * 9), q_seq, group)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("n_batch", [64, 65, 257])
def test_numbers_of_sequences(dtype, packed, n_batch):
    """Up to 64 sequences a wavefront scans them alone; equal lengths, and one that differs."""
    _check(P.Case(44, dtype, packed, n_batch, 1, 64, 16, [40] * n_batch), 1, 4)
    _check(P.Case(45, dtype, packed, n_batch, 1, 64, 16, [40] * (n_batch - 1) + [700]), 9, 2)
    _check(P.Case(46, dtype, packed, n_batch, 1, 64, 16, [0] * (n_batch - 1) + [700]), 2, 1)


@pytest.mark.parametrize("dtype,packed", KINDS)
def test_pages_longer_than_the_sequences(dtype, packed):
    """A page holds more than a step, the last step of a sequence ends in it; the table's other entries
    name no page."""
    _check(P.Case(47, dtype, packed, 3, 2, 64, 1024, [1, 700, 1030]), 3, 5)
    _check(P.Case(48, dtype, packed, 2, 2, 128, 512, [511, 513], max_pages=7), 1, 8)


def test_nothing_but_empty_sequences():
    for lens in ([0], [0, 0, 0], [-5, 0] * 40):
        _check(P.Case(49, "bf16", False, len(lens), 2, 64, 16, lens), 2, 3)


@pytest.mark.parametrize("dtype,packed", KINDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_seq,group", [(150, 2), (64, 3), (129, 1)])
def test_chunks_of_padded_sequences(dtype, packed, causal, q_seq, group):
    """Row blocks whose tokens see a part of the keys, or that hold none of the sequence's tokens; sequences
    with fewer rows than they bring tokens."""
    lens, new_rows = [150, 333, 90, 40, 0], [q_seq, 70, 1, 60, q_seq]
    _check(P.Case(50, dtype, packed, 5, 4, 64, 32, lens), q_seq, group, causal, new_rows)
    _check(P.Case(51, dtype, packed, 2, 1, 128, 16, [1000, 400]), q_seq, group, causal, [q_seq, 33])
