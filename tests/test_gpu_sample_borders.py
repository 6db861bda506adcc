"""sample_symbols where the draw is delicate: entries without a weight beside the border, small
numbers, weights and log-probabilities to the last bit that is promised.

A log-probability is log(w / total) in 64 bits, rounded once to float32.  Its 64-bit error: weights
are exp of (x - m) / T with three roundings of the exponent and a few of the series, which move the
total by at most 3 (log V + 1) 2^-53 of it, the sums add at most 60 roundings, the difference and the
logarithm three, and an exponent of z three of |z|: below 2^-46 (1 + |z|) in all."""
import math

import numpy as np
import pytest
import torch

import answering_oracle as ao
import optimized_transducer_amd as ot

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SMALL = 1e-30  # a min_p that takes the kernels with cuts and cuts nothing here

# who works on a row: (V, settings); entries beyond those of a test are -inf
PATHS = {"batch": (256, {}), "batch, two chunks": (512, {}), "wave": (256, {"min_p": SMALL}),
         "4 waves": (2000, {}), "8 waves": (8000, {"min_p": SMALL}), "16 waves": (16000, {}),
         "few": (2000, {"top_k": 512}), "few of a long row": (20000, {"top_k": 512}),
         "read in every step": (20000, {"min_p": SMALL}), "top_k of a row read in every step": (20000, {"top_k": 600}),
         "slices": (40000, {}), "slices, min_p": (40000, {"min_p": SMALL})}


def _to_device(x, V, dtype, device):
    """x (rows, n) at the front of rows of V, the rest -inf."""
    full = torch.full((x.shape[0], V), -math.inf, dtype=DT[dtype], device=device)
    full[:, :x.shape[1]] = torch.from_numpy(x.astype(np.float32)).to(device).to(DT[dtype])
    return full


def _check_log_prob(got, z, total):
    """got (float32) of entries at exponent z with weights of `total` remaining."""
    want = z - np.log(total)
    tol = 2.0 ** -24 * np.abs(want) + 2.0 ** -46 * (1 + np.abs(z))
    assert (np.abs(got.astype(np.float64) - want) <= tol).all()


def _two_halves(rng, rows, vec):
    """Rows of 64 lanes of `vec` entries, lanes 32-63 the entries of lanes 0-31 again: half of the
    weights lies in front of lane 32.  From a random lane on the end of each half is empty."""
    half = rng.standard_normal((rows, 32, vec)) * 2
    half[np.arange(32)[None, :] >= rng.integers(20, 32, rows)[:, None]] = -np.inf
    return np.concatenate([half, half], 1).reshape(rows, 64 * vec)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("path", list(PATHS))
def test_the_draw_never_leaves_what_remains(path, dtype, device):
    """u = 1/2 falls on the border between two halves of equal weights with masked entries around it:
    the answer is one of the two entries at the border, never a masked one."""
    V, settings = PATHS[path]
    rows, vec = 4000 if V <= 2000 else 1000, 4 if dtype == "f32" else 8
    V = max(V, 64 * vec)
    x = _two_halves(np.random.default_rng(V), rows, vec)
    t = _to_device(x, V, dtype, device)
    x = t[:, :64 * vec].double().cpu().numpy()
    symbols, log_probs = ot.sample_symbols(t, torch.full((rows,), 0.5, device=device), **settings)
    s, lp = symbols.cpu().numpy(), log_probs.cpu().numpy()
    n = 32 * vec
    last = n - 1 - np.argmax(np.isfinite(x[:, :n])[:, ::-1], 1)
    first = n + np.argmax(np.isfinite(x[:, n:]), 1)
    at = np.arange(rows)
    assert (np.isfinite(x[at, np.clip(s, 0, 64 * vec - 1)]) & (s >= 0) & (s < 64 * vec)).all()
    assert ((s == last) | (s == first)).all()
    m = x.max(1)
    _check_log_prob(lp, x[at, s] - m, np.exp(x - m[:, None]).sum(1))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [256, 2000, 20000])
def test_the_draw_never_takes_what_min_p_has_cut(V, dtype, device):
    """The same with entries that min_p leaves out in place of masked ones, with and without top_k."""
    vec = 4 if dtype == "f32" else 8
    V = max(V, 64 * vec)
    rows = 4000 if V <= 2000 else 500
    x = _two_halves(np.random.default_rng(V + 1), rows, vec)
    x[np.isneginf(x)] = -60.0
    t = _to_device(x, V, dtype, device)
    x = t[:, :64 * vec].double().cpu().numpy()
    u = torch.full((rows,), 0.5, device=device)
    n = 32 * vec
    last = n - 1 - np.argmax((x > -50)[:, :n][:, ::-1], 1)
    first = n + np.argmax((x > -50)[:, n:], 1)
    for settings in ({}, {"top_k": 64 * vec}):
        s, lp = (a.cpu().numpy() for a in ot.sample_symbols(t, u, min_p=1e-12, **settings))
        assert ((s == last) | (s == first)).all()
        m = x.max(1)
        w = np.where(x > -50, np.exp(x - m[:, None]), 0.0)
        _check_log_prob(lp, x[np.arange(rows), s] - m, w.sum(1))


@pytest.mark.parametrize("settings", [{}, {"min_p": SMALL}], ids=["no cuts", "min_p"])
def test_the_border_between_slices(settings, device):
    """Slices of 8192 entries, the second 32 of a row as the first, the end of each half empty, and
    u = 1/2: the last entry in front of the border or the first behind it, not any other of its slice."""
    rng = np.random.default_rng(64)
    rows, V = 100, 64 * 8192
    at = np.sort(rng.choice(8192, (32, 5), replace=False), 1)
    half = rng.standard_normal((rows, 32, 5)).astype(np.float32) * 2
    half[np.arange(32)[None, :] >= rng.integers(12, 32, rows)[:, None]] = -np.inf
    t = torch.full((rows, 64, 8192), -math.inf, device=device)
    where = torch.from_numpy(at).to(device).expand(rows, 32, 5)
    h = torch.from_numpy(half).to(device)
    t[:, :32].scatter_(2, where, h)
    t[:, 32:].scatter_(2, where, h)
    symbols, log_probs = ot.sample_symbols(t.view(rows, V), torch.full((rows,), 0.5, device=device), **settings)
    s = symbols.cpu().numpy()
    end = np.isfinite(half[:, :, 0]).sum(1) - 1  # the last slice of a half
    last = end * 8192 + at[end, 4]
    first = 32 * 8192 + at[0, 0]
    assert ((s == last) | (s == first)).all(), s[(s != last) & (s != first)][:5]
    m = half.reshape(rows, -1).max(1).astype(np.float64)
    x = np.where(s == last, half[np.arange(rows), end, 4], half[:, 0, 0])
    _check_log_prob(log_probs.cpu().numpy(), x - m,
                    2 * np.exp(half.reshape(rows, -1).astype(np.float64) - m[:, None]).sum(1))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("path", list(PATHS))
def test_small_numbers_find_small_entries_before_a_large_one(path, dtype, device):
    """Entries of weights around 1e-17 in front of one of weight 1, in the same 16 bytes and before
    them: numbers in the middle of each one's share draw it."""
    V, settings = PATHS[path]
    vec = 4 if dtype == "f32" else 8
    V = max(V, 64 * vec)
    x, u, want = [], [], []
    for base in (0, vec, 5 * vec, 17 * vec, 63 * vec, V // (2 * vec) * vec, (V // vec - 1) * vec):
        for places in ((0, 1, 2), (0, 1, vec - 1), (1, vec - 2, vec - 1)):
            row = np.full(V, -np.inf)
            row[base + np.array(places)] = (-38.5, -40.0, 0.0)
            if base > 0:
                row[base - 1], row[base // 2] = -39.0, -40.5
            at = np.nonzero(np.isfinite(row))[0]
            run = np.cumsum(np.exp(row[at]))
            for k in range(len(at)):
                number = np.float32(((run[k - 1] if k else 0.0) + run[k]) / 2 / run[-1])
                x.append(row)
                u.append(number)
                want.append(at[k])
    t = _to_device(np.stack(x), V, dtype, device)
    s, lp = ot.sample_symbols(t, torch.from_numpy(np.array(u, np.float32)).to(device), **settings)
    got, want = s.cpu().numpy(), np.array(want)
    assert np.array_equal(got, want), [(i, got[i], want[i]) for i in np.nonzero(got != want)[0][:5]]
    x = np.stack(x)
    _check_log_prob(lp.cpu().numpy(), x[np.arange(len(x)), want], np.exp(x).sum(1))


# (x, T, u): a row (x, 0) at temperature T, where u is less than 5e-15 of it below the first entry's
# share 1 / (1 + exp(-x / T)), which 64 bits tell apart by ten roundings or more
CLOSE = [("-0x1.a8fdb2p+1", 1.375, "0x1.501af8p-4"), ("-0x1.feaf5ep+0", 0.640625, "0x1.5c74d2p-5"),
         ("-0x1.feaf5ep+1", 1.28125, "0x1.5c74d2p-5"), ("-0x1.acbf0ap-1", 2.421875, "0x1.a85b28p-2"),
         ("-0x1.a8fdb2p+0", 0.6875, "0x1.501af8p-4"), ("-0x1.b44cb4p+1", 0.578125, "0x1.67893ap-9")]


@pytest.mark.parametrize("path", list(PATHS))
def test_weights_are_those_of_64_bits(path, device):
    """Numbers a few roundings of 64 bits away from the border between two entries."""
    V, settings = PATHS[path]
    x = np.full((len(CLOSE), V), -np.inf, np.float32)
    for i, (v, _, _) in enumerate(CLOSE):
        x[i, 17 * i] = float.fromhex(v)
        x[i, V // 2 + i] = 0.0
    T = torch.tensor([t for _, t, _ in CLOSE], device=device)
    u = torch.tensor([float.fromhex(n) for _, _, n in CLOSE], device=device)
    s, _ = ot.sample_symbols(_to_device(x, V, "f32", device), u, temperature=T, **settings)
    assert s.tolist() == [17 * i for i in range(len(CLOSE))]
    above = torch.nextafter(u, torch.ones_like(u))
    s, _ = ot.sample_symbols(_to_device(x, V, "f32", device), above, temperature=T, **settings)
    assert s.tolist() == [V // 2 + i for i in range(len(CLOSE))]


@pytest.mark.parametrize("V,settings", [(50, {}), (500, {}), (500, {"min_p": 0.01}), (1000, {"top_p": 0.9}),
                                        (3001, {}), (5000, {"top_k": 200, "top_p": 0.95}), (15000, {"top_p": 0.8}),
                                        (30000, {"top_k": 700}), (50000, {}), (50000, {"top_p": 0.9, "min_p": 1e-4})])
@pytest.mark.parametrize("temperature", [1.0, 0.3, 7.0])
def test_log_probs_are_rounded_once(V, settings, temperature, device):
    """The logarithm of 64 bits, rounded to float32: rows from flat to one entry of nearly all."""
    rng = np.random.default_rng(V)
    rows = 600 if V <= 5000 else 60
    x = (rng.standard_normal((rows, V)) * rng.choice([0.1, 1, 3, 10], (rows, 1))).astype(np.float32)
    x[:, 0] += rng.choice([0.0, 5.0, 15.0, 25.0], rows).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    s, lp = ot.sample_symbols(torch.from_numpy(x).to(device), torch.from_numpy(u).to(device),
                              temperature=temperature, **settings)
    s, lp = s.cpu().numpy(), lp.cpu().numpy()
    top_k, top_p, min_p = settings.get("top_k", 0), settings.get("top_p", 1.0), settings.get("min_p", 0.0)
    T = np.float64(np.float32(temperature))
    z, total = np.zeros(rows), np.zeros(rows)
    for r in range(rows):
        want, _ = ao.sample_row(x[r], float(u[r]), temperature, top_k, top_p, min_p)
        assert want == s[r]
        row = (x[r].astype(np.float64) - x[r].max()) / T
        w = np.sort(np.exp(row))[::-1]
        if top_k:
            w = w[:top_k]
        if top_p < 1:
            run = np.cumsum(w)
            w = w[:max(1, int((np.concatenate([[0.0], run[:-1]]) < np.float64(np.float32(top_p)) * run[-1]).sum()))]
        total[r] = math.fsum(w[w >= np.float64(np.float32(min_p))])
        z[r] = row[s[r]]
    _check_log_prob(lp, z, total)


def _near(rng, V):
    """An entry of weight 1, the others within 2e-6 of weight 0.52: sums of 32 bits round every one of
    them the same way."""
    x = (math.log(0.52) + 1e-6 * rng.random(V)).astype(np.float32)
    x[V // 3] = 0.0
    return x, 1.0


def _clusters(rng, V):
    """Two thirds of the weights, nearly equal ones, in one bin of 256 between the largest entry and
    the smallest, and a third in another: more of them than 32-bit sums count."""
    x = rng.random(V, dtype=np.float32)
    x[rng.random(V) < 1 / 3] -= np.float32(10.0)
    x[V // 5] = 1000.0
    return x, 1e6


@pytest.mark.parametrize("make,V,top_p", [(_near, 700001, 0.5), (_near, 700001, 0.9), (_clusters, 700001, 0.6),
                                          (_clusters, 30000001, 0.6), (_clusters, 30000001, 0.9)])
def test_top_p_where_sums_of_32_bits_are_far_off(make, V, top_p, device):
    """Rows of a workgroup each, of many near weights: the cut is found in a bounded number of passes."""
    x, T = make(np.random.default_rng(V), V)
    u = np.array([0.3, 0.999], np.float32)
    t = torch.from_numpy(x).to(device)
    s, lp = ot.sample_symbols(t.expand(2, V), torch.from_numpy(u).to(device), temperature=T, top_p=top_p)
    z = (x.astype(np.float64) - x.max()) / T
    w = np.exp(z)
    order = np.sort(x)[::-1]
    run = np.cumsum(np.exp((order.astype(np.float64) - x.max()) / T))
    n = int(np.searchsorted(run, np.float64(np.float32(top_p)) * run[-1])) + 1  # entries that remain
    kept = x > order[n - 1]
    at = np.nonzero(x == order[n - 1])[0]
    kept[at[:n - int(kept.sum())]] = True
    run = np.cumsum(np.where(kept, w, 0.0))
    want = [int(np.searchsorted(run, float(v) * run[-1], side="right")) for v in u]
    assert s.tolist() == want
    want_lp = z[want] - math.log(run[-1])
    assert (np.abs(lp.double().cpu().numpy() - want_lp) <= 2.0 ** -24 * np.abs(want_lp) + 2.0 ** -30).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [16385, 50000, 131072])
def test_slices_with_settings_of_each_row(V, dtype, device):
    """Rows in slices, each with a temperature, top_p and min_p of its own: greedy rows, rows without
    cuts, rows of every one of them, rows without an answer."""
    rng = np.random.default_rng(V)
    rows = 40
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
    x[::7, 0] += 12.0  # nearly all of a row in one entry
    x[5] = -np.inf
    x[9, V - 2] = np.nan
    t = torch.from_numpy(x).to(device).to(DT[dtype])
    x = t.float().cpu().numpy()
    u = rng.random(rows).astype(np.float32)
    u[12] = np.nan
    T = rng.choice([0.0, 0.4, 1.0, 1.7, -1.0, math.nan], rows).astype(np.float32)
    p = rng.choice([0.0, 0.3, 0.9, 0.999, 1.0, 4.0, math.nan], rows).astype(np.float32)
    q = rng.choice([0.0, 1e-3, 0.2, 1.0, math.nan], rows).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(device)  # noqa: E731
    s, lp = ot.sample_symbols(t, dev(u), temperature=dev(T), top_p=dev(p), min_p=dev(q))
    want, want_lp = ao.sample(x, u, T, 0, np.where(np.isnan(p), 1.0, p), np.where(np.isnan(q), 0.0, q))
    assert np.array_equal(s.cpu().numpy(), want)
    lp = lp.double().cpu().numpy()
    fine = np.isfinite(want_lp)
    assert np.array_equal(lp[~fine], want_lp[~fine])
    assert (np.abs(lp - want_lp)[fine] <= 2.0 ** -24 * np.abs(want_lp[fine]) + 2.0 ** -35).all()
    for settings in (dict(temperature=dev(T), top_p=0.9), dict(top_p=dev(p)), dict(temperature=0.8, min_p=dev(q)),
                     dict(temperature=dev(T), top_p=0.5, min_p=dev(q))):
        host = {"temperature": 1.0, "top_p": 1.0, "min_p": 0.0}
        host.update({k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in settings.items()})
        host = {k: np.where(np.isnan(v), {"temperature": 0.0, "top_p": 1.0, "min_p": 0.0}[k], v) for k, v in host.items()}
        s, _ = ot.sample_symbols(t, dev(u), **settings)
        assert np.array_equal(s.cpu().numpy(), ao.sample(x, u, top_k=0, **host)[0]), list(settings)
