"""The page pool's attempts: changes that belong together are made or taken back together."""
import numpy as np
import pytest

from test_paged_refusals import _pool, _sound


def _state(p):
    return p._host.tolist(), p._uses.tolist(), list(p._free), list(p._end), list(p._begin), dict(p._changed)


def test_attempt():
    p = _pool()
    p.grow([(0, 40), (1, 16)])
    p.share(2, 0, 32)
    before = _state(p)
    for change in (lambda: p.release(0), lambda: (p.release(1), p.release(2), p.release(0)), lambda: p.trim(0, 40),
                   lambda: p.grow([(3, 90)]), lambda: (p.release(2), p.share(2, 0, 40)), lambda: p.share(3, 2, 20)):
        for error in (RuntimeError, ValueError, KeyboardInterrupt):
            with pytest.raises(error):
                with p.attempt():
                    change()
                    raise error
            assert _state(p) == before
            _sound(p)
    with pytest.raises(RuntimeError, match="exhausted"):
        with p.attempt():
            p.release(1)
            p.grow([(1, 112), (3, 60)])
    assert _state(p) == before
    with p.attempt():
        p.release(1)
        p.grow([(1, 100)])
    assert p.held(1) == 7 and p.free_pages == 0
    with pytest.raises(ValueError):  # outside an attempt nothing is taken back
        p.grow([(2, 200)])
    _sound(p)


def test_random_attempts():
    """Groups of random changes, half of which fail: the pool is as before, the order of its free pages too."""
    rng = np.random.default_rng(2)
    p = _pool(pages=40, slots=8, cap=200)
    for _ in range(1500):
        before = _state(p)
        try:
            with p.attempt():
                for _ in range(rng.integers(1, 8)):
                    s, t = (int(x) for x in rng.choice(8, 2, replace=False))
                    op = rng.integers(5)
                    if op == 0:
                        p.release(s)
                    elif op == 1:
                        n = int(rng.integers(0, 200))
                        p.release(s)
                        if p.has(t, n):
                            p.share(s, t, n)
                    elif op == 2:
                        p.trim(s, int(rng.integers(0, 150)), int(rng.integers(0, 20)))
                    else:
                        p.grow([(s, int(rng.integers(1, 200))), (t, int(rng.integers(1, 60)))])
                if rng.integers(2):
                    raise RuntimeError
        except RuntimeError:
            assert _state(p) == before
        _sound(p)


def test_rehearsal():
    """Without keep nothing stays, and what the pool has no pages for is found."""
    p = _pool()
    p.grow([(0, 40), (1, 16)])
    before = _state(p)
    with p.attempt(keep=False):
        p.grow([(0, 100)])
        p.trim(0, 60)
        p.grow([(2, 80)])
        assert p.held(0) == 4 and p.held(2) == 5
    assert _state(p) == before
    with pytest.raises(RuntimeError, match="exhausted"):
        with p.attempt(keep=False):
            p.grow([(0, 100)])
            p.grow([(2, 80)])
    assert _state(p) == before
    _sound(p)
