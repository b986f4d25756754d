"""Seeds of the counter-based dropout modules that are given none: every module has one of
its own, positioned by counter_dropout_seed; given seeds stay as they are."""

import pytest


@pytest.fixture
def nn():
    import pyneural
    yield pyneural.nn
    pyneural.counter_dropout_seed(0)


def test_default_seeds_differ(nn):
    a, b, c = nn.CounterDropout(0.1), nn.CounterDropout(0.1), nn.CounterDropout(0.3, offset=5)
    assert len({a.seed, b.seed, c.seed}) == 3
    assert min(a.seed, b.seed, c.seed) >= 1 << 32  # apart from small seeds given by hand
    assert (a.offset, b.offset, c.offset) == (0, 0, 5)


def test_given_seeds_stay(nn):
    assert [nn.CounterDropout(0.1, seed=s).seed for s in (0, 7, 2 ** 64 - 1)] == [0, 7, 2 ** 64 - 1]
    assert nn.CounterDropout(0.1, 3, 4).seed == 3


def test_positioned(nn):
    runs = []
    for n in (0, 1, 0, (1 << 32) - 2):
        nn.counter_dropout_seed(n)
        runs.append([nn.CounterDropout(0.1).seed for _ in range(3)])
    assert runs[0] == runs[2] and not set(runs[0]) & set(runs[1])
    assert runs[1] == [(2 << 32) + k for k in range(3)]
    assert all(s < 1 << 64 for s in runs[3])
    for bad in (-1, (1 << 32) - 1, 1 << 40):
        with pytest.raises(ValueError):
            nn.counter_dropout_seed(bad)
