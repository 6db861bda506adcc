"""Answering with a joiner in 8 bits on the device: block quantisation, the projection of its
blocks and symbols drawn from logits, against 64-bit forms.

Tolerances.  Quantisation is defined bit for bit: values and scales are equal.  A projected logit
is a float32 sum of D products (each exact: 4-bit significands) and, per block, one scale product
and one fused multiply-add: at most 128 + 3 * blocks + 2 roundings of 2^-24 of the terms'
magnitude, plus half a step of the stored type.  A denominator moves by no more than the largest
error of its row's logits, plus 2^-22 for each exponential and merge on its way and one rounding.
Symbols are equal; a log-probability has a total of weights within 2^-22 each, and one rounding of
its own.  In 16 bits half a step is eps / 2: fp16 2^-11, bf16 2^-8."""
import math

import numpy as np
import pytest
import torch

import answering_oracle as ao
import optimized_transducer_amd as ot

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ---------------------------------------------------------------- quantisation
def _check_quantize(x, block_rows):
    values, scale = ot.quantize_blocks(x, block_rows)
    assert values.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    want_v, want_s = ao.quantize_blocks(x.float().cpu().numpy(), block_rows)
    assert values.shape == x.shape and scale.shape == want_s.shape
    np.testing.assert_array_equal(scale.cpu().numpy(), want_s)
    np.testing.assert_array_equal(values.float().cpu().numpy(), want_v.astype(np.float32))
    return values, scale


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 128), (3, 7), (2, 127), (5, 129), (127, 136), (128, 128), (129, 256),
                                    (300, 500), (1000, 512), (33, 1000), (2, 4096), (257, 2000), (200, 513), (131, 1021),
                                    (3, 4095)])
def test_quantize(rows, D, dtype, block_rows, device):
    rng = np.random.default_rng(rows * 31 + D)
    x = torch.from_numpy((rng.standard_normal((rows, D)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32))
    _check_quantize(x.to(DT[dtype]).to(device), block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_extremes(dtype, block_rows, device):
    """Zero blocks, subnormal and huge blocks, NaN and infinities that reach no other block."""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((300, 640)).astype(np.float32)
    x[0:128, 0:128] = 0
    x[:, 128:256] *= np.float32(1e-40)
    x[128:256, 256:384] *= np.float32(8e37)
    x[0, 300] = np.inf
    x[200, 500] = np.nan
    x[5, 520] = -0.0
    x[256:, 512:] *= np.float32(2.0 ** -120)
    t = torch.from_numpy(x).to(DT[dtype]).to(device)
    values, scale = _check_quantize(t, block_rows)
    # (one product above overflows to an infinity in float32 too): bad scales where bad entries are
    bad = ~torch.isfinite(t).cpu().numpy()
    bad = np.pad(bad, ((0, -300 % block_rows), (0, 0))).reshape(-1, block_rows, 5, 128).any((1, 3))
    assert bad.sum() >= 2 and np.array_equal(~torch.isfinite(scale).cpu().numpy(), bad)


def test_quantize_every_quotient_rounds_like_ieee(device):
    """All bfloat16 values of some binades against many maxima: quotients at and beside the
    midpoints of e4m3."""
    bits = np.arange(0x3E80, 0x4080, dtype=np.uint32) << 16
    v = bits.view(np.float32)
    rows = []
    for i in range(0, len(v), 4):
        r = np.concatenate([v[:127] * np.float32(0.5), v[i:i + 1] * np.float32(4)])
        rows.append(r)
        rows.append(np.concatenate([-v[300:427], v[i:i + 1] * np.float32(8)]))
    x = torch.from_numpy(np.stack(rows)).to(device)
    _check_quantize(x, 1)
    _check_quantize(x * 1.1754e-38, 1)
    _check_quantize(x * 3e-31, 1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_strides(dtype, device):
    rng = np.random.default_rng(4)
    big = torch.from_numpy(rng.standard_normal((300, 700)).astype(np.float32)).to(DT[dtype]).to(device)
    for view in (big[:, :512], big[3:, 1:513], big[::2, 8:264], big.t(), big[:1, 5:300], big[5:6].expand(9, 700),
                 big[:, 3:4]):
        for block_rows in (1, 128):
            v, s = ot.quantize_blocks(view, block_rows)
            v2, s2 = ot.quantize_blocks(view.contiguous(), block_rows)
            assert torch.equal(v.view(torch.uint8), v2.view(torch.uint8)) and torch.equal(s, s2)
            assert v.is_contiguous()


# ------------------------------------------------------------------ projection
def _operands(rng, rows, D, V, device, bias=True, spread=1.0):
    """Values and scales made on the host: every 8-bit value occurs, scales are any float32."""
    vals = np.concatenate([ao.E4M3, -ao.E4M3])
    x = vals[rng.integers(0, len(vals), (rows, D))]
    w = vals[rng.integers(0, len(vals), (V, D))]
    nb = -(-D // 128)
    xs = (np.exp(rng.standard_normal((rows, nb)) * spread) / 448).astype(np.float32)
    ws = (np.exp(rng.standard_normal((-(-V // 128), nb)) * spread) / 448 / math.sqrt(D)).astype(np.float32)
    b = rng.standard_normal(V).astype(np.float32) if bias else None
    t = lambda a: torch.from_numpy(a.astype(np.float32)).to(device)  # noqa: E731
    args = [t(x).to(torch.float8_e4m3fn), t(xs), t(w).to(torch.float8_e4m3fn), t(ws), None if b is None else t(b)]
    return args, (x, xs, w, ws, b)


def _check_project(args, host, dtype, denominators=True):
    x, xs, w, ws, b = host
    logits, den = ot.project_joiner_fp8(*args, logits_dtype=dtype, denominators=denominators)
    assert logits.dtype == dtype and logits.shape == (x.shape[0], w.shape[0])
    want, mag = ao.project(x, xs, w, ws, b)
    nb = xs.shape[1]
    tol = (128 + 3 * nb + 2) * 2.0 ** -24 * mag + 1e-37
    got = logits.double().cpu().numpy()
    stored = tol + STEP[dtype] * (np.abs(want) + tol) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    fits = np.abs(want) < torch.finfo(dtype).max * (1 - 2.0 ** -8)
    assert (np.abs(got - want) <= stored)[fits].all(), (np.abs(got - want) / stored)[fits].max()
    assert fits.mean() > 0.99
    if not denominators:
        assert den is None
        return logits, den
    m = want.max(1)
    ref = m + np.log(np.exp(want - m[:, None]).sum(1))
    d = den.double().cpu().numpy()
    dtol = tol.max(1) + (16 + -(-w.shape[0] // 64)) * 2.0 ** -22 + 2.0 ** -23 * np.abs(ref)
    assert (np.abs(d - ref) <= dtol).all(), (np.abs(d - ref) / dtol).max()
    return logits, den


SHAPES = [(1, 16, 1), (1, 128, 64), (2, 144, 5), (15, 64, 17), (16, 512, 500), (17, 512, 500), (32, 512, 500),
          (33, 1008, 131), (64, 256, 128), (65, 256, 129), (127, 128, 255), (128, 384, 256), (129, 640, 257),
          (1, 1024, 4096), (7, 2048, 1111), (300, 512, 500), (513, 192, 1030), (1003, 1008, 777), (2000, 512, 512),
          (1, 4096, 33), (257, 80, 4999), (4100, 112, 96),
          # each kernel at its smallest and odd sizes: blocks 1 to 4, then longer rows
          (13000, 16, 33), (13000, 128, 65), (6600, 240, 127), (3300, 256, 250), (3301, 384, 251), (3333, 400, 129),
          (1700, 512, 1021), (1700, 496, 1022), (6500, 1040, 257), (2111, 640, 1001), (5000, 2064, 130),
          (700, 1536 + 16, 3001),
          # enough tiles of 128 x 128 for the longer rows
          (9000, 1040, 1025), (16500, 640, 514), (2000, 528, 4997)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,D,V", SHAPES)
def test_project(rows, D, V, dtype, device):
    args, host = _operands(np.random.default_rng(rows * 7 + D + V), rows, D, V, device)
    logits, _ = _check_project(args, host, DT[dtype])
    # without the denominators: the same logits, bit for bit
    again, none = ot.project_joiner_fp8(*args, logits_dtype=DT[dtype], denominators=False)
    assert none is None and torch.equal(again.view(torch.uint8), logits.view(torch.uint8))


@pytest.mark.parametrize("rows,D,V", [(3, 256, 40), (300, 512, 300), (2000, 128, 500)])
def test_project_without_bias_and_with_scales_far_apart(rows, D, V, device):
    args, host = _operands(np.random.default_rng(9), rows, D, V, device, bias=False, spread=6.0)
    _check_project(args, host, torch.float32)


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_project_masked_entries(rows, device):
    """A bias of -inf masks entries out of the denominators; all of them masked leave -inf."""
    args, host = _operands(np.random.default_rng(11), rows, 256, 300, device)
    bias = args[4].clone()
    bias[100:] = -math.inf
    logits, den = ot.project_joiner_fp8(*args[:4], bias)
    want, _ = ao.project(*host[:4], None)
    assert torch.isneginf(logits[:, 100:]).all()
    y = want[:, :100] + args[4].double().cpu().numpy()[:100]
    ref = np.log(np.exp(y - y.max(1, keepdims=True)).sum(1)) + y.max(1)
    assert np.abs(den.double().cpu().numpy() - ref).max() <= 1e-3
    logits, den = ot.project_joiner_fp8(*args[:4], torch.full_like(bias, -math.inf))
    assert torch.isneginf(logits).all() and torch.isneginf(den).all()


@pytest.mark.parametrize("rows", [2, 500])
def test_project_a_bad_scale_stays_in_its_row_or_block(rows, device):
    args, host = _operands(np.random.default_rng(12), rows, 256, 300, device)
    clean, clean_den = ot.project_joiner_fp8(*args)
    xs, ws = args[1].clone(), args[3].clone()
    xs[1, 1] = math.nan
    logits, den = ot.project_joiner_fp8(args[0], xs, *args[2:])
    assert torch.isnan(logits[1]).all() and torch.isnan(den[1])
    keep = torch.arange(rows, device=device) != 1
    assert torch.equal(logits[keep], clean[keep]) and torch.equal(den[keep], clean_den[keep])
    ws[1, 0] = math.nan
    logits, _ = ot.project_joiner_fp8(*args[:3], ws, args[4])
    assert torch.isnan(logits[:, 128:256]).all()
    assert torch.equal(logits[:, :128], clean[:, :128]) and torch.equal(logits[:, 256:], clean[:, 256:])


def test_project_rows_do_not_depend_on_their_neighbours(device):
    """A row of a long batch is the row of a short one, within the bound; the same call gives the
    same bits."""
    rng = np.random.default_rng(13)
    args, host = _operands(rng, 3000, 512, 500, device)
    logits, den = ot.project_joiner_fp8(*args)
    again, den2 = ot.project_joiner_fp8(*args)
    assert torch.equal(logits, again) and torch.equal(den, den2)
    few, _ = ot.project_joiner_fp8(args[0][:5].contiguous(), args[1][:5].contiguous(), *args[2:])
    _, mag = ao.project(*(h[:5] if i < 2 else h for i, h in enumerate(host)))
    assert (np.abs((few - logits[:5]).cpu().numpy()) <= 2 * 142 * 2.0 ** -24 * mag).all()


# -------------------------------------------------------------------- sampling
def _check_sample(x, u, **settings):
    """x (rows, V) and u on the device; settings as sample_symbols takes them."""
    symbols, log_probs = ot.sample_symbols(x, u, **settings)
    assert symbols.dtype == torch.int32 and log_probs.dtype == torch.float32
    host = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    host.update({k: v.cpu().numpy() if torch.is_tensor(v) else v for k, v in settings.items()})
    want, want_lp = ao.sample(x.float().cpu().numpy(), u.cpu().numpy(), **host)
    got, got_lp = symbols.cpu().numpy(), log_probs.double().cpu().numpy()
    bad = np.nonzero(got != want)[0]
    assert not len(bad), (bad[:5], got[bad[:5]], want[bad[:5]])
    fine = np.isfinite(want_lp)
    assert np.array_equal(got_lp[~fine], want_lp[~fine])
    assert (np.abs(got_lp - want_lp)[fine] <= 2.0 ** -21 + 2.0 ** -23 * np.abs(want_lp[fine])).all()
    return symbols, log_probs


def _logits(rng, rows, V, dtype, device, sigma=3.0, masked=True, steps=None):
    x = rng.standard_normal((rows, V)).astype(np.float32) * np.float32(sigma)
    if steps:
        x = np.round(x * steps) / np.float32(steps)
    if masked and V > 4:
        x[:, V - V // 8:] = -np.inf
        x[rng.random((rows, V)) < 0.05] = -np.inf
    if masked and rows > 3:
        x[rows // 2] = -np.inf
    u = rng.random(rows, dtype=np.float32)
    return torch.from_numpy(x).to(DT[dtype]).to(device), torch.from_numpy(u).to(device)


SETTINGS = {"none": {}, "temperature": {"temperature": 0.6}, "greedy": {"temperature": 0.0}, "top_k": {"top_k": 7},
            "top_1": {"top_k": 1}, "top_p": {"top_p": 0.8}, "top_p_0": {"top_p": 0.0}, "min_p": {"min_p": 0.05},
            "all": {"temperature": 1.3, "top_k": 40, "top_p": 0.9, "min_p": 0.01},
            "wide": {"temperature": 4.0, "top_k": 400, "top_p": 0.97}}


@pytest.mark.parametrize("settings", list(SETTINGS))
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 255, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2047, 4100, 5000])
def test_sample(V, settings, device):
    rng = np.random.default_rng(V)
    for dtype in DT:
        x, u = _logits(rng, 37, V, dtype, device)
        _check_sample(x, u, **SETTINGS[settings])


@pytest.mark.parametrize("settings", ["none", "greedy", "top_k", "top_p", "all", "wide"])
@pytest.mark.parametrize("V", [8191, 16384, 33333, 65537, 131072, 200001])
def test_sample_long_rows(V, settings, device):
    rng = np.random.default_rng(V)
    for dtype in DT:
        x, u = _logits(rng, 5, V, dtype, device, sigma=2.0)
        _check_sample(x, u, **SETTINGS[settings])


@pytest.mark.parametrize("rows,V", [(1, 500), (3000, 32), (2111, 500), (1500, 777), (700, 1500)])
def test_sample_many_rows(rows, V, device):
    rng = np.random.default_rng(rows)
    x, u = _logits(rng, rows, V, "f32", device)
    for s in ("none", "all"):
        _check_sample(x, u, **SETTINGS[s])


@pytest.mark.parametrize("rows,V", [(300, 16400), (257, 50000), (3, 524288), (2, 524289), (129, 33000)])
def test_sample_long_rows_in_batches(rows, V, device):
    """More rows than slices are kept for at a time, the longest row that is cut into slices, the next one."""
    rng = np.random.default_rng(rows)
    x, u = _logits(rng, rows, V, "bf16", device, sigma=1.5)
    for settings in ({}, {"top_p": 0.9}, {"min_p": 0.2}, {"temperature": 2.0, "top_p": 0.99, "min_p": 1e-3}):
        _check_sample(x, u, **settings)


@pytest.mark.parametrize("V", [20000, 70000])
def test_sample_long_rows_of_few_values(V, device):
    """Cuts inside thousands of equal values, next to rows of two values one rounding apart."""
    rng = np.random.default_rng(V)
    x = rng.integers(0, 3, (8, V)).astype(np.float32)
    x[4:] = np.nextafter(np.float32(7), np.float32(8) * rng.integers(0, 2, (4, V)).astype(np.float32))
    x[6, rng.random(V) < 0.9] = -np.inf
    x[7] = -30.0
    x[7, V - 3] = 5.0
    x = torch.from_numpy(x).to(device)
    u = torch.from_numpy(rng.random(8, dtype=np.float32)).to(device)
    for p in (0.0, 1e-6, 0.3, 0.5, 0.9, 1.0 - 2.0 ** -24):
        _check_sample(x, u, top_p=p)
        _check_sample(x, u, top_p=p, temperature=1e-3)
        _check_sample(x, u, top_p=p, temperature=1e6, min_p=0.999999)


def test_sample_a_long_row_does_not_depend_on_its_neighbours(device):
    rng = np.random.default_rng(8)
    x, u = _logits(rng, 300, 20000, "f32", device)
    for s in ({"top_p": 0.8}, {"top_p": 0.95, "min_p": 0.01, "temperature": 1.4}):
        a, lp = ot.sample_symbols(x, u, **s)
        for r in (0, 1, 255, 256, 299):
            b, lq = ot.sample_symbols(x[r:r + 1], u[r:r + 1], **s)
            assert int(b) == int(a[r]) and float(lq) == float(lp[r])
        again, lq = ot.sample_symbols(x, u, **s)
        assert torch.equal(a, again) and torch.equal(lp, lq)


@pytest.mark.parametrize("V", [64, 500, 1100, 6000, 40000])
def test_sample_ties(V, device):
    """Values on a coarse grid: the cuts of top_k and top_p fall inside runs of equal values."""
    rng = np.random.default_rng(V + 1)
    for steps in (1, 4):
        x, u = _logits(rng, 24, V, "bf16", device, steps=steps)
        for k in (1, 3, V // 10 + 1, V - 1, V, V + 5):
            _check_sample(x, u, top_k=k)
            _check_sample(x, u, top_k=k, top_p=0.7, temperature=2.0)
        for p in (0.1, 0.35, 0.9, 0.999):
            _check_sample(x, u, top_p=p)


@pytest.mark.parametrize("V", [64, 512, 1024, 4096, 32768])
def test_sample_borders_that_sums_hit_exactly(V, device):
    """Equal entries: sums are whole numbers, and u * total and top_p * total fall on them."""
    x = torch.full((65, V), 2.5, device=device)
    u = torch.arange(65, device=device) / 64.0
    got, lp = _check_sample(x, u)
    want = (torch.arange(65, device=device) * (V // 64)).clamp(max=V - 1)
    assert torch.equal(got.long(), want)
    for p in (0.25, 0.5, 0.75):
        got, _ = _check_sample(x, u, top_p=p)
        assert int(got.max()) == int(V * p) - 1
    _check_sample(x, u, top_k=V // 2, top_p=0.5)
    x[:, ::2] = -1e4  # weights of exactly zero in between
    _check_sample(x, u)
    _check_sample(x, u, top_p=0.5)


@pytest.mark.parametrize("V", [7, 300, 2000, 20000])
def test_sample_small_weights_and_border_numbers(V, device):
    """u = 0 takes the first entry with any weight at all, however small; u of 1 and above the last."""
    rng = np.random.default_rng(V)
    x = rng.standard_normal((12, V)).astype(np.float32)
    x[:4] *= 100
    x[4:8] *= 20
    x = torch.from_numpy(x).to(device)
    for v in (0.0, -1.0, 1.0 - 2.0 ** -24, 1.0, 2.0, 2.0 ** -24, 1e-38):
        u = torch.full((12,), v, device=device)
        _check_sample(x, u)
        _check_sample(x, u, top_k=5, top_p=0.9)
    u = torch.full((12,), math.nan, device=device)
    s, lp = ot.sample_symbols(x, u)
    assert (s == -1).all() and torch.isneginf(lp).all()


@pytest.mark.parametrize("V", [9, 512, 3001, 12345])
def test_sample_rows_without_an_answer_and_extremes(V, device):
    rng = np.random.default_rng(V)
    x = rng.standard_normal((10, V)).astype(np.float32)
    x[0] = -np.inf
    x[1, V // 2] = np.nan
    x[2, V - 1] = np.inf
    x[3] = -np.inf
    x[3, V - 2] = -3e38
    x[4] = 3e38
    x[5, ::2] = -3e38
    x[5, 1::2] = 3e38
    x[6] = 0.0
    x[6, ::3] = -0.0
    x[7, 0] = -np.nan
    x[8] = 1e-42 * np.arange(V)
    t = torch.from_numpy(x).to(device)
    u = torch.from_numpy(rng.random(10, dtype=np.float32)).to(device)
    for settings in ({}, {"temperature": 0.0}, {"temperature": 1e-30}, {"temperature": math.inf}, {"top_k": 3},
                     {"top_p": 0.5}, {"min_p": 1.0}, {"temperature": 1e30, "top_k": 5, "top_p": 0.6, "min_p": 0.2}):
        s, _ = _check_sample(t, u, **settings)
        assert s[[0, 1, 2, 7]].tolist() == [-1] * 4 and int(s[3]) == V - 2


@pytest.mark.parametrize("V", [100, 500, 1030, 5000, 50000])
def test_sample_settings_of_each_row(V, device):
    rng = np.random.default_rng(V)
    rows = 60 if V < 10000 else 12
    x, u = _logits(rng, rows, V, "f32", device)
    dev = lambda a, t: torch.from_numpy(a.astype(t)).to(device)  # noqa: E731
    t = rng.choice([0.0, 0.3, 1.0, 2.0, -1.0, math.nan], rows)
    k = rng.choice([0, 1, 5, V // 3, V + 9, -4], rows)
    p = rng.choice([0.0, 0.2, 0.9, 1.0, 7.0, -2.0], rows)
    m = rng.choice([0.0, 0.01, 1.0, 3.0, -1.0], rows)
    _check_sample(x, u, temperature=dev(t, np.float32), top_k=dev(k, np.int32), top_p=dev(p, np.float32),
                  min_p=dev(m, np.float32))
    # one tensor among numbers
    _check_sample(x, u, temperature=0.7, top_k=dev(k, np.int32), top_p=0.9)
    nan = torch.full((rows,), math.nan, device=device)
    a = ot.sample_symbols(x, u, top_p=nan, min_p=nan)
    b = ot.sample_symbols(x, u)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sample_strides(dtype, device):
    rng = np.random.default_rng(2)
    for V, W in ((500, 512), (501, 700), (64, 65), (3000, 3007), (20000, 20001)):
        big = torch.from_numpy(rng.standard_normal((21, W)).astype(np.float32)).to(DT[dtype]).to(device)
        u = torch.rand(21, device=device)
        for view, n in ((big[:, :V], u), (big[:, W - V:], u), (big[::3, :V], u[::3]), (big[:, :V].flip(0), u),
                        (big[2:3, :V].expand(21, V), u)):
            for s in ("none", "all"):
                a = ot.sample_symbols(view, n, **SETTINGS[s])
                b = ot.sample_symbols(view.contiguous(), n.contiguous(), **SETTINGS[s])
                assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        _check_sample(big[:, :V], u, top_p=0.9)
    t = torch.from_numpy(rng.standard_normal((90, 21)).astype(np.float32)).to(DT[dtype]).to(device).t()
    _check_sample(t, u, top_k=9)


def test_sample_a_row_does_not_depend_on_its_neighbours(device):
    rng = np.random.default_rng(6)
    x, u = _logits(rng, 5000, 500, "f32", device)
    for s in ("none", "all"):
        a, lp = ot.sample_symbols(x, u, **SETTINGS[s])
        for r in (0, 1, 2499, 4999):
            b, lq = ot.sample_symbols(x[r:r + 1], u[r:r + 1], **SETTINGS[s])
            assert int(b) == int(a[r]) and float(lq) == float(lp[r])


# ------------------------------------------------------------------ all of them
def test_no_rows(device):
    v, s = ot.quantize_blocks(torch.zeros((0, 512), device=device))
    assert v.shape == (0, 512) and s.shape == (0, 4)
    assert ot.quantize_blocks(torch.zeros((0, 130), device=device), 128)[1].shape == (0, 2)
    w, ws = ot.quantize_blocks(torch.ones((500, 512), device=device), 128)
    logits, den = ot.project_joiner_fp8(v, s, w, ws)
    assert logits.shape == (0, 500) and den.shape == (0,)
    symbols, lp = ot.sample_symbols(logits, torch.zeros(0, device=device))
    assert symbols.shape == (0,) and lp.shape == (0,)


def test_refusals(device):
    f8 = torch.zeros((2, 128), device=device).to(torch.float8_e4m3fn)
    one = torch.ones((2, 1), device=device)
    w1 = torch.ones((1, 1), device=device)
    x, u = torch.zeros((2, 5), device=device), torch.zeros(2, device=device)
    for match, call in [
            ("block_rows must be 1 or 128", lambda: ot.quantize_blocks(x, 64)),
            ("shape", lambda: ot.quantize_blocks(u)),
            ("D > 0", lambda: ot.quantize_blocks(torch.zeros((2, 0), device=device))),
            ("expect x", lambda: ot.project_joiner_fp8(f8, one, f8[:, :64], w1)),
            ("multiple of 16", lambda: ot.project_joiner_fp8(f8[:, :100], one, f8[:, :100], w1)),
            ("V > 0", lambda: ot.project_joiner_fp8(f8, one, f8[:0], w1[:0])),
            ("x_scale must have shape", lambda: ot.project_joiner_fp8(f8, w1, f8, w1)),
            ("weight_scale must have shape", lambda: ot.project_joiner_fp8(f8, one, f8, one)),
            ("contiguous", lambda: ot.project_joiner_fp8(f8[:, :64], one, f8[:, :64], w1)),
            ("one HIP device", lambda: ot.project_joiner_fp8(f8, one.cpu(), f8, w1)),
            ("bias must have shape", lambda: ot.project_joiner_fp8(f8, one, f8, w1, u[:1])),
            ("logits_dtype must be", lambda: ot.project_joiner_fp8(f8, one, f8, w1, logits_dtype=torch.float64)),
            ("shape", lambda: ot.sample_symbols(u, u)),
            ("V > 0", lambda: ot.sample_symbols(x[:, :0], u)),
            ("uniform must be", lambda: ot.sample_symbols(x, u[:1])),
            ("uniform must be", lambda: ot.sample_symbols(x, u.double())),
            ("uniform must be", lambda: ot.sample_symbols(x, u.cpu())),
            ("temperature must be >= 0", lambda: ot.sample_symbols(x, u, temperature=-1.0)),
            ("temperature must be >= 0", lambda: ot.sample_symbols(x, u, temperature=math.nan)),
            ("top_k must be >= 0", lambda: ot.sample_symbols(x, u, top_k=-1)),
            ("top_p must be in", lambda: ot.sample_symbols(x, u, top_p=1.1)),
            ("top_p must be in", lambda: ot.sample_symbols(x, u, top_p=math.nan)),
            ("min_p must be in", lambda: ot.sample_symbols(x, u, min_p=-0.1)),
            ("temperature must be a number or", lambda: ot.sample_symbols(x, u, temperature=u.double())),
            ("top_k must be a number or", lambda: ot.sample_symbols(x, u, top_k=u)),
            ("top_p must be a number or", lambda: ot.sample_symbols(x, u, top_p=u[:1])),
            ("min_p must be a number or", lambda: ot.sample_symbols(x, u, min_p=u.cpu()))]:
        with pytest.raises(RuntimeError, match=match):
            call()


def test_streams_do_not_share_anything(device):
    """Two streams, each with its own batch, in turn without waiting for each other."""
    rng = np.random.default_rng(8)
    work = []
    for i in range(2):
        args, _ = _operands(rng, 700 + 300 * i, 512, 500, device)
        x, u = _logits(rng, 900, 1200 + i, "f32", device)
        work.append((args, x, u))
    want = [(ot.project_joiner_fp8(*a), ot.sample_symbols(x, u, top_p=0.9)) for a, x, u in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (a, x, u) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append((ot.project_joiner_fp8(*a), ot.sample_symbols(x, u, top_p=0.9)))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            for a, b in zip(g[0] + g[1], want[i][0] + want[i][1]):
                assert torch.equal(a, b)


def _step(enc, dec, one, zero, w, ws, bias, u):
    """One decoding step: the joiner's activations of each stream, its logits, a symbol."""
    x = ot.pack_joiner(enc, dec, one, zero, activation="tanh", out_dtype=torch.bfloat16)
    q, s = ot.quantize_blocks(x)
    logits, den = ot.project_joiner_fp8(q, s, w, ws, bias)
    return (logits, den) + ot.sample_symbols(logits, u, temperature=0.8, top_p=0.95)


def test_decoding_step_end_to_end(device):
    """pack_joiner -> quantize_blocks -> project_joiner_fp8 -> sample_symbols, each stage against
    its 64-bit form on the stage before."""
    rng = np.random.default_rng(20)
    N, D, V = 32, 512, 500
    t = lambda a: torch.from_numpy(a.astype(np.float32)).to(device)  # noqa: E731
    enc, dec = t(rng.standard_normal((N, 1, D))), t(rng.standard_normal((N, 1, D)))
    one = torch.ones(N, dtype=torch.int32, device=device)
    w, ws = ot.quantize_blocks(t(rng.standard_normal((V, D)) * 4 / math.sqrt(D)), 128)
    bias, u = t(rng.standard_normal(V)), torch.rand(N, device=device)
    logits, den, symbols, lp = _step(enc, dec, one, torch.zeros_like(one), w, ws, bias, u)
    x = torch.tanh(enc + dec).to(torch.bfloat16)[:, 0]
    packed = ot.pack_joiner(enc, dec, one, torch.zeros_like(one), activation="tanh", out_dtype=torch.bfloat16)
    assert (packed.float() - x.float()).abs().max() <= 2.0 ** -7  # a step of bfloat16 near 1
    q, s = _check_quantize(packed, 1)
    host = [q.double().cpu().numpy(), s.cpu().numpy(), w.double().cpu().numpy(), ws.cpu().numpy(), bias.cpu().numpy()]
    again, den2 = _check_project([q, s, w, ws, bias], host, torch.float32)
    assert torch.equal(again, logits) and torch.equal(den, den2)
    s2, lp2 = _check_sample(logits, u, temperature=0.8, top_p=0.95)
    assert torch.equal(s2, symbols) and torch.equal(lp2, lp)


def test_scoring_with_the_denominators(device):
    """A batch scored with the 8-bit projection: the loss from its denominators is the loss from
    its float32 logits alone."""
    rng = np.random.default_rng(21)
    T, U = np.array([30, 17, 1, 22]), np.array([9, 0, 3, 12])
    rows, D, V = int((T * (U + 1)).sum()), 256, 500
    args, _ = _operands(rng, rows, D, V, device)
    i32 = lambda a: torch.from_numpy(a.astype(np.int32)).to(device)  # noqa: E731
    targets = i32(rng.integers(1, V, (4, 12)))
    logits, den = ot.project_joiner_fp8(*args)
    with torch.no_grad():
        a = ot.transducer_loss(logits, targets, i32(T), i32(U), 0, False, reduction="sum", denominators=den)
        b = ot.transducer_loss(logits, targets, i32(T), i32(U), 0, False, reduction="sum")
    # each of a path's T + U denominators within 1e-5 of the other
    assert abs(float(a) - float(b)) <= 1e-5 * float((T + U).sum())


def test_chain_replays_from_a_hip_graph(device):
    """quantize -> project -> sample captured once; every replay on new inputs is the eager call."""
    rng = np.random.default_rng(22)
    D, V, rows = 512, 500, 300
    t = lambda a: torch.from_numpy(a.astype(np.float32)).to(device)  # noqa: E731
    w, ws = ot.quantize_blocks(t(rng.standard_normal((V, D)) / 8), 128)
    bias = t(rng.standard_normal(V))
    x, u = torch.empty((rows, D), device=device), torch.empty(rows, device=device)
    temperature = torch.empty(rows, device=device)

    def chain(x, u, temperature):
        q, s = ot.quantize_blocks(x)
        logits, den = ot.project_joiner_fp8(q, s, w, ws, bias)
        return (logits, den) + ot.sample_symbols(logits, u, temperature=temperature, top_k=50, top_p=0.9)

    x.normal_()
    u.uniform_()
    temperature.fill_(1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(x, u, temperature)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same call
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(x, u, temperature))
        graphs.append(g)
    for i in range(6):
        x.normal_()
        u.uniform_()
        temperature.uniform_(0.0, 2.0)
        want = chain(x, u, temperature)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs[i % 2], want):
            assert torch.equal(a, b)
        torch.rand(1000, device=device).sum().item()


def test_sample_long_rows_replay_and_overlap(device):
    """Rows that several workgroups share: two graphs, and calls on two streams at once, do not share anything."""
    rows, V = 70, 60000
    x, u = torch.empty((rows, V), device=device), torch.empty(rows, device=device)
    draw = lambda x, u: ot.sample_symbols(x, u, temperature=0.9, top_p=0.9, min_p=1e-4)  # noqa: E731
    x.normal_()
    u.uniform_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        draw(x, u)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(draw(x, u))
        graphs.append(g)
    for i in range(6):
        x.normal_()
        u.uniform_()
        want = draw(x, u)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2][0], want[0]) and torch.equal(outs[i % 2][1], want[1])
        torch.rand(1000, device=device).sum().item()
    inputs = [(torch.randn((rows, V), device=device) * 2, torch.rand(rows, device=device)) for _ in range(2)]
    want = [draw(*i) for i in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(draw(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for a in got[k]:
            assert torch.equal(a[0], want[k][0]) and torch.equal(a[1], want[k][1])


def test_offsets_beyond_32_bits(device):
    """More than 2^32 elements of logits: the last rows are the rows of a small call."""
    rows, V = 70001, 65536  # 4.6e9 elements, 9.2 GB of bfloat16
    x = torch.empty((rows, V), dtype=torch.bfloat16, device=device)
    x.normal_()
    u = torch.rand(rows, device=device)
    a, lp = ot.sample_symbols(x, u)
    b, lq = ot.sample_symbols(x[-40:].clone(), u[-40:])
    assert torch.equal(a[-40:], b) and torch.equal(lp[-40:], lq)
    _check_sample(x[-3:], u[-3:])
    x8, s = ot.quantize_blocks(x)
    v8, t = ot.quantize_blocks(x[-40:].clone())
    assert torch.equal(x8[-40:].view(torch.uint8), v8.view(torch.uint8)) and torch.equal(s[-40:], t)
    x8, s = ot.quantize_blocks(x, 128)
    first = (rows - 40) // 128 * 128  # the last blocks of rows
    v8, t = ot.quantize_blocks(x[first:].clone(), 128)
    assert torch.equal(x8[first:].view(torch.uint8), v8.view(torch.uint8)) and torch.equal(s[first // 128:], t)


def test_project_offsets_beyond_32_bits(device):
    """Logits of more than 2^31 elements, 2^32 bytes."""
    g = torch.Generator(device=device).manual_seed(1)
    rows, D, V = 1050001, 128, 2100
    x8, s = ot.quantize_blocks(torch.randn((rows, D), device=device, generator=g).bfloat16())
    w, ws = ot.quantize_blocks(torch.randn((V, D), device=device, generator=g), 128)
    logits, den = ot.project_joiner_fp8(x8, s, w, ws, logits_dtype=torch.bfloat16)
    n = 1000
    few, den2 = ot.project_joiner_fp8(x8[-n:].clone(), s[-n:].clone(), w, ws, logits_dtype=torch.bfloat16)
    assert (logits[-n:].float() - few.float()).abs().max() <= 2.0 ** -6 * float(few.float().abs().max())
    assert (den[-n:] - den2).abs().max() <= 1e-3
    mid = rows // 2
    few, _ = ot.project_joiner_fp8(x8[mid:mid + n].clone(), s[mid:mid + n].clone(), w, ws, logits_dtype=torch.bfloat16)
    assert (logits[mid:mid + n].float() - few.float()).abs().max() <= 2.0 ** -6 * float(few.float().abs().max())
