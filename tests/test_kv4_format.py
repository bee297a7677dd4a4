"""The definition of the 4-bit cache's values (kv4_oracle), on the CPU: what the format
promises of a quantized row, and that words and rotations are what they say."""
import numpy as np
import pytest

from . import kv4_oracle as k4


def test_words():
    codes = np.arange(-8, 8).reshape(2, 8)
    assert [hex(w) for w in k4.pack(codes).view(np.uint32)[:, 0]] == ["0x75316420", "0xfdb9eca8"]
    x = np.random.default_rng(0).integers(-8, 8, (3, 5, 64))
    assert np.array_equal(k4.unpack(k4.pack(x)), x)


@pytest.mark.parametrize("size", [1.0, 1e-20, 1e25])
def test_a_row_is_off_by_half_a_step(size):
    """The largest of a group is code -8 of a step that is at most one scale above its eighth;
    what no code is past (the opposite end) is off by half a step."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((500, 96)) * np.exp(rng.normal(0, 1, (500, 96)))).astype(np.float32) * np.float32(size)
    codes, sub, bits = k4.quantize(x)
    scale = k4.bf16(bits).astype(np.float64)[:, None]
    g = x.reshape(500, 3, 32).astype(np.float64)
    most = np.abs(g).max(-1)
    n = np.abs(sub.astype(np.float64))
    assert n.min() >= 1 and n.max() == 127
    assert (n * scale * 8 >= most * (1 - 2.0 ** -23)).all() and (((n - 1) * scale * 8 < most) | (n == 1)).all()
    assert (scale[:, 0] * 127 * 8 >= most.max(-1) * (1 - 2.0 ** -23)).all()
    assert (scale[:, 0] * 127 * 8 <= most.max(-1) * (1 + 2.0 ** -7)).all()
    step = (sub * scale)[..., None]
    back = codes.reshape(500, 3, 32) * step
    assert codes.min() == -8 and np.abs(codes.reshape(500, 3, 32) * (most[..., None] == np.abs(g))).max() == 8
    inside = g / step <= 7.5
    assert (np.abs(back - g)[inside] <= np.abs(np.broadcast_to(step, g.shape))[inside] / 2 * (1 + 2.0 ** -50)).all()
    assert (np.abs(back - g) <= np.abs(step)).all()


def test_rows_at_the_ends():
    x = np.zeros((6, 32), np.float32)
    x[1, :3] = [1.0, -1.0, 0.5]                     # of two, the negative
    x[2, :4] = [np.inf, -np.inf, np.nan, 2.0]       # the finite one sets the step
    x[3, 5] = 1e-31                                 # below 2^-100
    x[4, :2] = [3e38, 1.0]                          # above 2^126
    x[5, :2] = [np.nan, np.inf]                     # nothing to set it
    codes, sub, bits = k4.quantize(x)
    assert (codes[0] == 0).all() and bits[0] == 0
    assert sub[1, 0] == 127 and list(codes[1, :3]) == [7, -8, 4]
    assert sub[2, 0] == -127 and list(codes[2, :4]) == [-8, 7, 0, -8]
    assert bits[3] == 0 and codes[4, 0] == -8 and np.isfinite(k4.bf16(bits[4])) and bits[5] == 0 and (codes[5] == 0).all()


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotation(neighbours):
    """A rotation by p + n is one by p and one by n; sizes stay; dims past the table's stay as they are."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 3, 64)).astype(np.float32)
    t = k4.table(50, 40)
    y = k4.rotate(x, np.array([0, 5, 17, 49]), t, neighbours)
    assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 40:], x[..., 40:])
    # one f32 rounding a value of y, and one of each cosine and sine: 2^-24 each of at most |a| + |b|
    assert np.allclose((y.astype(np.float64) ** 2).sum(-1), (x.astype(np.float64) ** 2).sum(-1), rtol=2.0 ** -20)
    z = k4.rotate(k4.rotate(x, np.full(4, 20), t, neighbours), np.full(4, 13), t, neighbours)
    assert np.abs(z - k4.rotate(x, np.full(4, 33), t, neighbours)).max() < 6 * 2.0 ** -24 * 2 * np.abs(x).max()
