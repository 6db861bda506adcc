"""The order of additions of a draw, without a GPU: where sums over lanes do not grow, and that a draw
does not leave the entries with a weight there."""
import numpy as np
import pytest

import answering_oracle as ao
import draw_model


def two_halves(rng, rows, vec):
    """Rows of 64 lanes of `vec` entries, lanes 32-63 the entries of lanes 0-31 again: half of the
    weights lies in front of lane 32.  From a random lane on the end of each half is empty."""
    half = rng.standard_normal((rows, 32, vec)) * 2
    half[np.arange(32)[None, :] >= rng.integers(20, 32, rows)[:, None]] = -np.inf
    return np.concatenate([half, half], 1).reshape(rows, 64 * vec).astype(np.float32)


@pytest.mark.parametrize("vec", [4, 8])
def test_scan_sums_the_lanes_in_front(vec):
    v = np.random.default_rng(0).integers(0, 1000, (50, 64)).astype(np.float64)
    assert np.array_equal(draw_model.scan(v), np.cumsum(v, 1))
    w = np.random.default_rng(1).integers(0, 9, (50, 64, vec)).astype(np.float64)
    assert np.array_equal(draw_model.pairwise(w), w.sum(2))


@pytest.mark.parametrize("vec", [4, 8])
def test_draw_stays_among_the_entries_with_a_weight(vec):
    """Targets between the sums of a lane with the last weight of a half and of an empty lane behind
    it: such rows are there, and each draws one of the two entries at the border."""
    rows, n = 3000, 32 * vec
    x = two_halves(np.random.default_rng(vec), rows, vec)
    w = draw_model.weights(x.astype(np.float64))
    upto = draw_model.scan(draw_model.pairwise(w))
    empty = w.sum(2) == 0
    target = 0.5 * upto[:, -1:]
    # the first lane whose sum passes the target is an empty one
    first = np.argmax(upto > target, 1)
    assert empty[np.arange(rows), first].sum() > 10
    got = draw_model.draw(w, np.full(rows, 0.5))
    front = n - 1 - np.argmax(np.isfinite(x[:, :n])[:, ::-1], 1)
    behind = n + np.argmax(np.isfinite(x[:, n:]), 1)
    assert ((got == front) | (got == behind)).all()


@pytest.mark.parametrize("vec", [4, 8])
def test_draw_is_the_oracles_away_from_borders(vec):
    rng = np.random.default_rng(10 + vec)
    x = (rng.standard_normal((300, 64 * vec)) * 3).astype(np.float32)
    x[rng.random(x.shape) < 0.3] = -np.inf
    u = rng.random(300, dtype=np.float32)
    got = draw_model.draw(draw_model.weights(x.astype(np.float64)), u.astype(np.float64))
    assert np.array_equal(got, ao.sample(x, u, 1.0, 0, 1.0, 0.0)[0])


@pytest.mark.parametrize("vec", [4, 8])
def test_draw_of_small_numbers(vec):
    """Entries of small weights in front of a large one in the same lane: their running sums are kept,
    which the difference of the lane's sum and its own would not."""
    for lane in (0, 1, 17, 63):
        x = np.full((1, 64 * vec), -np.inf)
        x[0, lane * vec + np.arange(3)] = (-38.5, -40.0, 0.0)
        if lane:
            x[0, 1] = -39.0
        w = draw_model.weights(x)
        at = np.nonzero(np.isfinite(x[0]))[0]
        run = np.cumsum(w.reshape(-1)[at])
        middle = (run + np.concatenate([[0.0], run[:-1]])) / 2 / run[-1]
        got = draw_model.draw(np.repeat(w, len(at), 0), middle)
        assert np.array_equal(got, at)


def test_search_for_the_cut_ends_at_it():
    rng = np.random.default_rng(5)
    values = [float(v) for v in (rng.standard_normal(400) * 3).astype(np.float32)] + [0.0, 1e-45, -1e-45]
    for cut in values[::7] + [0.0, 1e-45, -1e-45]:
        for start in (min(values), 0.0, max(values), values[17]):
            answer = lambda v: 0 if v == cut else 1 if v < cut else -1  # noqa: E731
            seen = draw_model.search(values, start, answer)
            assert seen[-1] == cut and len(seen) <= 40


@pytest.mark.parametrize("turn", [0.0, -1e-45, 1e-45, 0.3])
@pytest.mark.parametrize("far", [-5.0, 5.0])
def test_search_for_the_cut_ends_where_sums_contradict_each_other(turn, far):
    """Roundings can put the cut above one value and below the next, and at neither: the search ends
    there all the same, at a value of the row, around zero too, whose two signs are one value."""
    values = [float(v) for v in np.linspace(-6, 6, 200).astype(np.float32)] + [0.0, 1e-45, -1e-45]
    start = min(values) if far < 0 else max(values)
    for at_turn in (1, -1):
        answer = lambda v: 1 if v < turn else -1 if v > turn else at_turn  # noqa: E731
        seen = draw_model.search(values, start, answer)
        assert len(seen) <= 40 and seen[-1] in values
