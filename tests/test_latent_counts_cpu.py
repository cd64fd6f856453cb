"""The exact counts of oracle/latent.py see a tile that a long call loses or reads twice (no GPU)."""
import pytest
import torch

from oracle import latent as ol

BF, HF = torch.bfloat16, torch.float16


def _rounded(tokens, dtype):
    """What a kernel gives that read so many tokens of each tile."""
    o, lse, _, _ = ol.counted(tokens, dtype)
    return o.to(dtype)[None], lse.float()[None]


def _close(got, want):
    o, l, b_o, b_l = want
    ol.close(got[0], got[1], (o[None], l[None], b_o[None], b_l[None]))


# lengths of the GPU tests: cut requests, a long prefix, lists of several phases
LENGTHS = [(HF, 1300), (HF, 9000), (BF, 9000), (HF, 20000), (BF, 20000), (HF, 2293777)]


@pytest.mark.parametrize("dtype,n", LENGTHS)
def test_what_is_read_once_is_accepted(dtype, n):
    full = ol.whole(n)
    assert full.sum() == n and full[-1] == (n - 1) % 32 + 1
    _close(_rounded(full, dtype), ol.counted(full, dtype))


@pytest.mark.parametrize("dtype,n", LENGTHS)
@pytest.mark.parametrize("where", [0.0, 0.37, 0.5, 1.0])
def test_a_lost_or_doubled_tile_is_seen(dtype, n, where):
    full = ol.whole(n)
    at = int(where * (full.numel() - 2))  # a whole tile
    want = ol.counted(full, dtype)
    for times in (0, 2):
        bad = full.clone()
        bad[at] *= times
        with pytest.raises(AssertionError, match="out|lse"):
            _close(_rounded(bad, dtype), want)
        with pytest.raises(AssertionError):  # by the sum alone
            ol.close(want[0].to(dtype)[None], _rounded(bad, dtype)[1], tuple(x[None] for x in want))


@pytest.mark.parametrize("dtype,n", LENGTHS)
@pytest.mark.parametrize("other", [1, 2, 255, 256, 257, 512])
def test_a_tile_in_another_ones_place_is_seen(dtype, n, other):
    """As many tokens as there are, but one tile twice and another not at all: only o shows it."""
    full = ol.whole(n)
    at = (full.numel() // 2 - other) % (full.numel() - 1)
    to = (at + other) % (full.numel() - 1)
    if at == to:
        pytest.skip("not so many tiles")
    bad = full.clone()
    bad[at], bad[to] = 0, 64
    with pytest.raises(AssertionError, match="out"):
        _close(_rounded(bad, dtype), ol.counted(full, dtype))


@pytest.mark.parametrize("dtype,n,phase", [(HF, 2293777, 256), (HF, 2293777, 280), (BF, 20000, 64)])
def test_a_lost_phase_is_seen(dtype, n, phase):
    """Of each workgroup's tiles only the first described ones, as a list of several phases could lose."""
    full = ol.whole(n)
    keep = torch.arange(full.numel()) % phase < phase - 24
    with pytest.raises(AssertionError):
        _close(_rounded(full * keep, dtype), ol.counted(full, dtype))


def test_marks_name_their_tile():
    rows = torch.full((20000, 576), float("nan"), dtype=HF)
    ol.mark(rows)
    assert (rows[:, 512:] == 0).all() and (rows.sum(1) == 2).all()
    o, lse, _, _ = ol.attend(torch.zeros(1, 576), rows, rows[:, :512], 20000, 1.0, HF)
    want = ol.counted(ol.whole(20000), HF)
    # sums of 20000 terms in 64 bits, each partial sum within 2^-53 of itself and at most 1
    assert (o[0] - want[0]).abs().max() < 20002 * 2.0 ** -53 and abs(lse[0] - want[1]) < 20002 * 2.0 ** -53
