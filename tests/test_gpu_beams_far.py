"""Beam search's selection over large logits: a row's sum of exponentials goes by the largest number so far,
rounded below 2^16 and exact from there on, and moves from the one to the other within lanes, between the
lanes of a wave and between waves."""

import pytest
import torch

from tests import test_gpu_beams as beams_tests
from tests.test_gpu_beams import BF16, FP32, check
from tests.test_gpu_paged import banner

pytestmark = pytest.mark.gpu


def far_bound(vocab):
    """`bound_of`, and what moving a lane's sum costs: once in two of its pieces at most (512 numbers each, dealt to
    four waves) and once to its wave's largest number, each time a power of two (2^-23 of itself), a product
    (2^-24) and the argument's rounding, 2^-24 of a difference. The differences that a term passes add up to its
    own, of which `bound_of` counts three times 2^-24 where one is needed for the term itself."""
    return (8 * -(-vocab // 2048) + 48 + 3 * (-(-vocab // 4096) + 1)) * 2.0 ** -24


@pytest.fixture(autouse=True)
def bound(monkeypatch):
    monkeypatch.setattr(beams_tests, "bound_of", far_bound)


def scores_of(rows):
    return -(torch.arange(rows, device="cuda") % 5).float() / 4


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("rows,vocab", [(6, 8192), (6, 5001), (2052, 16384), (2052, 9003)])
def test_ramps(rows, vocab, dtype):
    """Numbers that rise or fall through all sizes from -10^5 to 10^5: every piece has a new largest number, or
    only the first has."""
    banner("ramps", rows, vocab, dtype)
    rise = torch.linspace(-1e5, 1e5, vocab, device="cuda")
    for row in (rise, -rise, rise - 1e5, rise / 1000 - 65586, rise / 1000 + 65486, rise.abs(), -rise.abs()):
        x = row.expand(rows, -1) + torch.arange(rows, device="cuda")[:, None] % 7
        check(x.to(dtype).contiguous(), scores_of(rows), 6, 9)


@pytest.mark.parametrize("near", [1e3, 6e4, 65536.0, 1e6, -1e3, -6e4, -65536.0, -1e6])
@pytest.mark.parametrize("rows,vocab", [(6, 4099), (2052, 8192)])
def test_close_together_far_out(near, rows, vocab):
    """Numbers a few units apart, so that all of them count, below 2^16, across it and beyond."""
    banner("close together", near, rows, vocab)
    gen = torch.Generator(device="cuda").manual_seed(int(abs(near)) + vocab)
    x = near + torch.randint(-24, 25, (rows, vocab), generator=gen, device="cuda").float() / 4
    check(x, scores_of(rows), 6, 12)
    # a cell, a wave's cells, or a lane's numbers on the other side, by what they are added to
    other = torch.full((rows, vocab), near, device="cuda")
    step = torch.arange(vocab, device="cuda")
    for on in (step // 512 % 2 == 0, step // 512 % 4 == 1, step // 8 % 64 < 32, step // 8 % 64 == 63, step < vocab // 2,
               step >= vocab // 2):
        check(torch.where(on, other + 3, other - 3), scores_of(rows), 6, 12)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_sizes_that_change_along_a_row(dtype):
    """Small numbers before far ones and behind them, up and down, 2048 rows that a wave reads by itself."""
    banner("changing sizes", dtype)
    rows, vocab = 2052, 32768
    gen = torch.Generator(device="cuda").manual_seed(3)
    noise = torch.randn(rows, vocab, generator=gen, device="cuda")
    for levels in ((0., 70000., 0., 65530.), (-70000., -65530., -65540., -65530.), (65530., 65540., 70000., 1e9),
                   (1e9, 70000., 65530., 0.), (-1e9, -70000., -65530., 0.), (3e38, -3e38, 3e38, 0.),
                   (-3e38, -1e9, -70000., -65540.)):
        level = torch.tensor(levels, device="cuda").repeat_interleave(vocab // 4)
        check((level + noise).to(dtype), scores_of(rows), 4, 8)
