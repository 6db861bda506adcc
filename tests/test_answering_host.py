"""The 8-bit answering operators without a GPU: the 64-bit forms the GPU tests compare with, the
refusals of the Python entry points that need no device, and those of the C ABI."""
import ctypes
import math

import numpy as np
import pytest
import torch

import answering_oracle as ao
import cabi
import optimized_transducer_amd as ot


def test_e4m3_values_are_torchs():
    q = np.concatenate([np.linspace(-448, 448, 20001), np.array([2.0 ** -10, 2.0 ** -9, 3 * 2.0 ** -10, 0.0]),
                        (ao.E4M3[1:] + ao.E4M3[:-1]) / 2]).astype(np.float32)
    want = torch.from_numpy(q).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(ao.to_e4m3(q), want)
    assert ao.E4M3[-1] == 448.0 and len(ao.E4M3) == 127


def test_quantize_oracle_rounds_to_the_nearest_value():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((37, 200)).astype(np.float32)
    for block_rows in (1, 128):
        v, s = ao.quantize_blocks(x, block_rows)
        back = v * np.repeat(np.repeat(s, block_rows, 0)[:37], 128, 1)[:, :200]
        scale = np.repeat(np.repeat(s, block_rows, 0)[:37], 128, 1)[:, :200]
        # half a step: 2^-4 of a normal value, 2^-10 scales below
        assert (np.abs(back - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * scale) * (1 + 1e-6)).all()
        assert np.abs(v).max() == 448.0


def test_sample_oracle_on_rows_worked_by_hand():
    x = np.log(np.array([1, 4, 2, 4, 1], np.float64)).astype(np.float32)
    draw = lambda u, t=1.0, k=0, p=1.0, q=0.0: ao.sample_row(x, u, t, k, p, q)[0]  # noqa: E731
    assert [draw(u) for u in (0.0, 0.08, 0.1, 0.5, 0.7, 0.95)] == [0, 0, 1, 2, 3, 4]
    assert [draw(u, k=2) for u in (0.0, 0.49, 0.51, 0.99)] == [1, 1, 3, 3]
    assert [draw(u, k=1) for u in (0.0, 0.99)] == [1, 1]          # the tie goes to the lower index
    assert [draw(u, p=0.5) for u in (0.0, 0.99)] == [1, 3]        # 4 < 6 <= 8
    assert [draw(u, p=0.7) for u in (0.0, 0.45, 0.99)] == [1, 2, 3]
    assert [draw(u, q=0.4) for u in (0.0, 0.45, 0.99)] == [1, 2, 3]
    assert draw(0.3, t=0.0) == 1 and draw(1.0) == 4 and draw(0.99, p=0.0) == 1
    assert ao.sample_row(np.full(4, -math.inf, np.float32), 0.5, 1, 0, 1, 0) == (-1, -math.inf)
    assert ao.sample_row(np.array([0, math.nan], np.float32), 0.5, 1, 0, 1, 0)[0] == -1


def test_sample_oracle_frequencies():
    rng = np.random.default_rng(1)
    x = rng.standard_normal(20).astype(np.float32)
    u = (np.arange(20000) + 0.5) / 20000
    got = np.bincount([ao.sample_row(x, v, 0.7, 0, 1.0, 0.0)[0] for v in u], minlength=20) / 20000
    want = np.exp(x / 0.7) / np.exp(x / 0.7).sum()
    assert np.abs(got - want).max() <= 1.0 / 20000 + 1e-6


def test_python_entry_points_refuse_before_touching_a_device():
    f8 = torch.zeros((2, 128), dtype=torch.float8_e4m3fn)
    one = torch.ones((2, 1))
    with pytest.raises(RuntimeError, match="must be on a HIP device"):
        ot.quantize_blocks(torch.zeros(2, 128))
    with pytest.raises(RuntimeError, match="must be float32, float16 or bfloat16"):
        ot.quantize_blocks(torch.zeros((2, 128), dtype=torch.float64))
    with pytest.raises(RuntimeError, match="has no gradient"):
        ot.quantize_blocks(torch.zeros((2, 128), requires_grad=True))
    with pytest.raises(RuntimeError, match="one HIP device"):
        ot.project_joiner_fp8(f8, one, f8, torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="must be float8_e4m3fn"):
        ot.project_joiner_fp8(torch.zeros(2, 128), one, f8, torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="scales must be float32"):
        ot.project_joiner_fp8(f8, one.half(), f8, torch.ones((1, 1)))
    with pytest.raises(RuntimeError, match="has no gradient"):
        ot.project_joiner_fp8(f8, one, f8, torch.ones((1, 1)), torch.zeros(2, requires_grad=True))
    with pytest.raises(RuntimeError, match="must be on a HIP device"):
        ot.sample_symbols(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(RuntimeError, match="must be float32, float16 or bfloat16"):
        ot.sample_symbols(torch.zeros((2, 5), dtype=torch.int32), torch.zeros(2))
    with pytest.raises(TypeError):
        ot.sample_symbols(torch.zeros(2, 5), torch.zeros(2), top_k=1.5)


def test_c_abi_refuses_bad_arguments():
    L = cabi.lib()
    null, one, odd = ctypes.c_void_p(0), ctypes.c_void_p(64), ctypes.c_void_p(65)
    i32, i64, f32, size = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_size_t
    L.ot_joiner_project_blocks_workspace_bytes.restype = size

    def quantize(x=one, dtype=0, stride=128, rows=4, D=128, block_rows=1, values=one, scale=one):
        return L.ot_quantize_blocks(x, i32(dtype), i64(stride), i64(rows), i32(D), i32(block_rows), values,
                                    scale, null)

    assert quantize(rows=0) == 0  # nothing to do
    for bad in (dict(x=null), dict(values=null), dict(scale=null), dict(rows=-1), dict(rows=1 << 31), dict(D=0),
                dict(D=-4), dict(stride=-1), dict(block_rows=64), dict(block_rows=0), dict(dtype=7),
                dict(D=2 ** 31 - 1)):
        assert quantize(**bad) == -1, bad
    for bad in (dict(x=odd), dict(scale=odd), dict(x=ctypes.c_void_p(66))):
        assert quantize(**bad) == -3, bad

    def project(x=one, xs=one, w=one, ws=one, bias=null, rows=4, D=128, V=10, logits=one, dtype=0, den=null,
                work=null, work_bytes=0):
        return L.ot_joiner_project_blocks(x, xs, w, ws, bias, i64(rows), i32(D), i32(V), logits, i32(dtype), den,
                                          work, size(work_bytes), null)

    assert project(rows=0) == 0
    for bad in (dict(x=null), dict(xs=null), dict(w=null), dict(ws=null), dict(logits=null), dict(rows=-1),
                dict(rows=1 << 31), dict(D=0), dict(D=120), dict(D=-16), dict(V=0), dict(V=-1), dict(dtype=9),
                dict(den=one), dict(den=one, work=one, work_bytes=8), dict(V=2 ** 31 - 1),
                dict(D=2 ** 31 - 16)):
        assert project(**bad) == -1, bad
    for bad in (dict(x=ctypes.c_void_p(72)), dict(w=ctypes.c_void_p(72)), dict(xs=odd), dict(ws=odd),
                dict(bias=odd), dict(logits=odd), dict(logits=ctypes.c_void_p(66)),
                dict(den=odd, work=one, work_bytes=1 << 20), dict(den=one, work=odd, work_bytes=1 << 20)):
        assert project(**bad) == -3, bad
    need = L.ot_joiner_project_blocks_workspace_bytes
    assert need(i64(0), i32(5)) == 0 and need(i64(5), i32(0)) == 0 and need(i64(5), i32(500)) > 0

    def sample(logits=one, dtype=0, stride=10, rows=4, V=10, uniform=one, t=null, k=null, p=null, m=null,
               symbols=one, log_probs=one, work=null, work_bytes=0):
        return L.ot_sample_symbols(logits, i32(dtype), i64(stride), i64(rows), i32(V), uniform, t, f32(1), k,
                                   i32(0), p, f32(1), m, f32(0), symbols, log_probs, work, size(work_bytes), null)

    assert sample(rows=0) == 0
    L.ot_sample_symbols_workspace_bytes.restype = size
    need = L.ot_sample_symbols_workspace_bytes
    assert need(i64(4), i32(500), i32(0)) == 0 and need(i64(0), i32(50000), i32(0)) == 0
    assert need(i64(4), i32(50000), i32(1)) == 0 and need(i64(4), i32(50000), i32(0)) > 0
    assert need(i64(1 << 20), i32(50000), i32(0)) == need(i64(256), i32(50000), i32(0))
    for bad in (dict(logits=null), dict(uniform=null), dict(symbols=null), dict(log_probs=null), dict(rows=-1),
                dict(rows=1 << 31), dict(V=0), dict(V=2 ** 31 - 1), dict(stride=-1), dict(dtype=5)):
        assert sample(**bad) == -1, bad
    # the indices of a step of 16 waves x 64 lanes x 8 elements past the end stay below 2^31
    assert sample(V=2 ** 31 - 8192) == -1 and sample(dtype=1, V=2 ** 31 - 4097) == -1
    assert sample(V=50000, work=odd, work_bytes=1 << 24) == -3
    for bad in (dict(logits=odd), dict(logits=ctypes.c_void_p(66)), dict(uniform=odd), dict(t=odd), dict(k=odd),
                dict(p=odd), dict(m=odd), dict(symbols=odd), dict(log_probs=odd)):
        assert sample(**bad) == -3, bad


@pytest.mark.parametrize("which", range(5))
def test_projection_refuses_every_operand_that_asks_for_a_gradient(which):
    f8 = lambda *shape: torch.zeros(shape, dtype=torch.float8_e4m3fn)  # noqa: E731
    args = [f8(2, 128), torch.ones(2, 1), f8(3, 128), torch.ones(1, 1), torch.zeros(3)]
    args[which].requires_grad_()
    with pytest.raises(RuntimeError, match="has no gradient"):
        ot.project_joiner_fp8(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="one HIP device"):
        ot.project_joiner_fp8(*args)
