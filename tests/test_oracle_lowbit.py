"""The CPU restatement of MX4 and of the 8-bit cache against known values (no GPU)."""
import numpy as np
import pytest

from oracle import lowbit as LB


def test_mx4_known_block():
    x = np.zeros((1, 32))
    x[0, :10] = [6.0, -6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.2]
    codes, scales = LB.mx4_quantize(x)
    assert scales.tolist() == [[127]]  # floor(log2 6) - 2 = 0
    nib = np.stack((codes & 15, codes >> 4), -1).reshape(-1)
    assert nib[:10].tolist() == [7, 15, 0, 2, 2, 4, 4, 6, 6, 8]  # ties to even codes, the sign kept
    assert np.array_equal(LB.mx4_decode(codes, scales)[0, :10], [6, -6, 0, 1, 1, 2, 2, 4, 4, 0])


@pytest.mark.parametrize("top,byte", [(0.0, 0), (1.0, 125), (7.9, 127), (8.0, 128), (2.0 ** -125, 0), (2.0 ** -140, 0),
                                      (3e38, 252), (np.inf, 255), (np.nan, 255)])
def test_mx4_scale_byte(top, byte):
    x = np.zeros((1, 5))
    x[0, 2] = top
    assert LB.mx4_quantize(x)[1].tolist() == [[byte]]


def test_mx4_saturates_and_round_trips():
    x = np.full((1, 32), 7.9)
    assert (LB.mx4_decode(*LB.mx4_quantize(x)) == 6).all()
    grid = np.concatenate([LB.E2M1, -LB.E2M1, LB.E2M1, -LB.E2M1])[None] * 2.0 ** -9
    assert np.array_equal(LB.mx4_decode(*LB.mx4_quantize(grid)), grid)


def test_e4m3_table_and_encoding():
    assert LB.E4M3[0x7E] == 448 and LB.E4M3[1] == 2.0 ** -9 and np.isnan(LB.E4M3[0x7F]) and LB.E4M3[0xFE] == -448
    fin = np.array([i for i in range(256) if i & 127 != 127])
    assert np.array_equal(LB.encode8(LB.E4M3[fin], "e4m3"), fin)
    assert LB.encode8(np.array([0.53125, 0.59375, 2.0 ** -10, 3 * 2.0 ** -10]), "e4m3").tolist() == [0x30, 0x32, 0, 2]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_grows_by_powers_of_two_and_stays_within_a_step(kind):
    """Many small growths: what is held stays within one step of the final scale."""
    rng = np.random.default_rng(3)
    codes, scales = np.zeros((1, 1, 64, 8), np.uint8), np.zeros((1, 1), np.float32)
    xs = rng.standard_normal((64, 1, 8)) * (1.06 ** np.arange(64))[:, None, None]
    for t in range(64):
        LB.append(xs[t:t + 1].astype(np.float32), codes, scales, np.zeros((1, 1), np.int32), [t + 1], [1], kind)
        assert np.log2(scales[0, 0]) % 1 == 0
    got = LB.decode8(codes[0, 0], kind) * scales[0, 0]
    step = scales[0, 0] if kind == "int8" else scales[0, 0] * np.maximum(2.0 ** -9, np.abs(got / scales[0, 0]) / 8)
    assert (np.abs(got - xs[:, 0]) <= step).all()


def test_append_first_slot_starts_the_scale_anew():
    codes, scales = np.full((1, 1, 16, 4), 77, np.uint8), np.full((1, 1), 1e6, np.float32)
    LB.append(np.full((1, 1, 4), 1.0), codes, scales, np.zeros((1, 1), np.int32), [1], [1], "int8")
    assert scales[0, 0] == 2.0 ** -6 and (codes[0, 0, 0] == 64).all() and (codes[0, 0, 1:] == 77).all()


def test_attention_uniform_and_empty_rows():
    rng = np.random.default_rng(0)
    c = rng.integers(0, 256, (2, 1, 16, 8), dtype=np.uint8)
    s = np.ones((2, 1), np.float32)
    q = np.zeros((3, 2, 8))
    o, _, _ = LB.attention(q, c, c, s, s, np.array([[1, 0]]), [2], [3], "int8", scale=1.0)
    v = LB.decode8(c, "int8")[1, 0]
    assert (o[0] == 0).all()  # position -1 sees nothing
    assert np.allclose(o[1], v[0]) and np.allclose(o[2], v[:2].mean(0))


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 9), (False, 0), (False, 12)])
def test_attention_of_all_rows_is_attention_row_by_row(causal, window):
    rng = np.random.default_rng(window)
    k, v = (rng.integers(-127, 128, (9, 2, 16, 8)).astype(np.int8).view(np.uint8) for _ in range(2))
    ks, vs = (rng.uniform(-0.02, 0.03, (9, 2)).astype(np.float32) for _ in range(2))
    table, lengths, counts = rng.permutation(9)[:8].reshape(2, 4).astype(np.int32), [50, 3], [7, 5]
    table[0, 1], table[1, 1:] = -1, -1
    args = (rng.standard_normal((12, 6, 8)), k, v, ks, vs, table, lengths, counts, "int8")
    a = LB.attention(*args, scale=0.3, causal=causal, window=window)
    b = LB.attention_of_all(*args, scale=0.3, causal=causal, window=window)
    for x, y in zip(a, b):
        assert np.allclose(x, y, rtol=1e-12, atol=1e-14)
