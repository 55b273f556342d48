"""Outputs that lie over inputs which other CTAs still read are refused on the host, before anything is launched (every call here is refused:
the addresses are no memory)."""
import pytest

from flashrt_b200 import _lib

A = 1 << 20                                                # stands for an aligned device pointer; never read
INVALID = -1


def softmax(out, rows=4, vocab=100, istride=100, ostride=100, flags=2):
    return _lib.call_status("frt_b200_softmax_rows", A, istride, out, ostride, None, rows, vocab, flags, None)


def verify(out, n=6):
    return _lib.call_status("frt_b200_verify_drafts", A + 4096, 100, None, 100, A, A + 8192, A + 8448, A + 8704, A + 8960, out, A + 9216, A + 9472, n, 2, 100,
                            0, None)


def plan(lens, batch=8):
    return _lib.call_status("frt_b200_paged_plan", A, A + 1024, A + 4096, 8, A + 8192, A + 16384, A + 16388, A + 16640, lens, None, None, None, 6, batch, 16, 16,
                            0, None)


@pytest.mark.parametrize("flags,row", [(2, 400), (0, 200)])
def test_probabilities(flags, row):
    for at in (0, 4, row, 4 * row - 4, -4, -1596):         # four rows of logits, four of probabilities of 400 bytes
        assert softmax(A + at, flags=flags) == INVALID, at
    wide = 1000 // (4 if flags else 2)                     # both in rows of 1000 bytes: 100 values of the one reach into the other
    for at in (0, row - 4, 604, 1000 + row - 4, -396, 3000 + row - 4, -3396):
        assert softmax(A + at, istride=wide, ostride=250, flags=flags) == INVALID, at
    for at in (0, row - 4, -396, 420):                     # rows of other steps, 1000 and 500 bytes; at last, the second over the second
        assert softmax(A + at, istride=wide, ostride=125, rows=3, flags=flags) == INVALID, at


def test_verification():
    for at in (0, 4, 20, -4, -20):
        assert verify(A + at) == INVALID, at


def test_plan():
    for at in (0, 4, 28, -28, 1024, 1024 + 28, 1024 - 28):
        assert plan(A + at) == INVALID, at
