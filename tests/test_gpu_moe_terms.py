"""What a mixture-of-experts layer hands from its gated product h to the output product: all of h, for numbers up to the largest, and infinities as such.
One expert without activation, so that h = (x gate) (x up) is known to the bit and rows of `down` with a single one give it back."""
import numpy as np
import pytest

from test_gpu_moe_scales import run

pytestmark = pytest.mark.gpu

ONE, MINUS = 2, 8  # the codes of 1.0 and of a sign


def parts(hidden, inter):
    shape = {"gate": (inter, hidden), "up": (inter, hidden), "down": (hidden, inter)}
    return {n: np.zeros(s, np.uint8) for n, s in shape.items()}, {n: np.full((s[0], s[1] // 32), 127, np.uint8) for n, s in shape.items()}


@pytest.mark.parametrize("tokens", (1, 20, 40))
@pytest.mark.parametrize("gate,up,exponent", ((4095, 4097, 104),   # the largest number
                                             (4095, 4096, 104),
                                             (4088, 4096, 104),    # 2^128 - 2^119, halfway between the largest bf16 value and 2^128
                                             (4087, 4096, 104), (4095, 4097, 103), (4095, 4097, 90)))
def test_h_up_to_the_largest_number(gpu, tokens, gate, up, exponent):
    """x = (4096, 1, 1, ...): gate = 4096 - 1 - ..., up = 4096 + 1 or 4096, with their scales 2^52."""
    hidden = inter = 32
    codes, scales = parts(hidden, inter)
    x = np.zeros((tokens, hidden), np.float32)
    x[:, 0], x[:, 1:16] = 4096.0, 1.0
    codes["gate"][:, 0], codes["gate"][:, 1:1 + 4096 - gate] = ONE, ONE | MINUS
    codes["up"][:, 0], codes["up"][:, 1:1 + up - 4096] = ONE, ONE
    codes["gate"][::3, 0] ^= MINUS  # -4096 - ...: negated as a whole
    codes["gate"][::3, 1:1 + 4096 - gate] ^= MINUS
    codes["down"][np.arange(hidden), np.arange(hidden)] = ONE
    scales["gate"][:], scales["up"][:] = 127 + exponent // 2, 127 + exponent - exponent // 2
    want = np.ldexp(np.float64(gate * up), exponent) * np.where(np.arange(inter) % 3 == 0, -1.0, 1.0)
    got = run(gpu, x, codes, scales, hidden, inter)
    assert np.array_equal(got.astype(np.float64), np.tile(want, (tokens, 1)))


@pytest.mark.parametrize("tokens", (1, 20, 40))
def test_an_infinite_h_makes_infinities(gpu, tokens):
    """h[5] = +-inf, the others numbers; every value of `down` is other than zero, so its sign is y's."""
    hidden, inter = 96, 64
    rng = np.random.default_rng(tokens)
    codes, scales = parts(hidden, inter)
    x = np.zeros((tokens, hidden), np.float32)
    x[:, 0] = np.where(np.arange(tokens) % 2 == 0, 2.0, -2.0)
    codes["gate"][:, 0] = codes["up"][:, 0] = ONE
    scales["gate"][5], scales["up"][5] = 127 + 64, 127 + 63  # 2^65 2^64
    codes["up"][5, 0] |= MINUS
    codes["down"][:] = rng.integers(1, 8, size=codes["down"].shape) | rng.choice(np.array([0, MINUS]), size=codes["down"].shape)
    got = run(gpu, x, codes, scales, hidden, inter)
    want = np.where(codes["down"][:, 5] & MINUS, np.inf, -np.inf)
    assert np.array_equal(got, np.tile(want, (tokens, 1)).astype(np.float32))


def cut(h, terms):
    """What `terms` bf16 values, rounded to the nearest one after the other, hold of whole numbers h."""
    kept, rest = np.zeros(h.shape), h.astype(np.float64)
    for _ in range(terms):
        m, e = np.frexp(rest)
        term = np.ldexp(np.rint(m * 256), e - 8)
        kept, rest = kept + term, rest - term
    return kept


@pytest.mark.parametrize("exponent", (0, 60, -120, -133))  # of h's last bit: 2^-133 is the smallest that bf16 has
@pytest.mark.parametrize("tokens,hidden,inter", ((1, 32, 32), (5, 64, 96), (33, 96, 288), (50, 32, 1056)))
def test_all_bits_of_h_arrive(gpu, tokens, hidden, inter, exponent):
    """h = (x gate) (x up) of small whole numbers, up to 24 bits; a row of `down` gives back one of its columns, times 1 or -1, to the bit. (Two terms would
    not do: checked on the host.)"""
    rng = np.random.default_rng(inter + tokens)
    codes, scales = parts(hidden, inter)
    whole = np.array([0, 2, 4, 5, 6], np.uint8)  # 0, 1, 2, 3, 4
    for name in ("gate", "up"):
        codes[name][:] = rng.choice(whole, size=codes[name].shape) | rng.choice(np.array([0, MINUS], np.uint8), size=codes[name].shape)
    value = {2: 1, 4: 2, 5: 3, 6: 4, 0: 0}
    w = {n: np.vectorize(lambda c: value[c & 7] * (-1 if c & 8 else 1))(codes[n]).astype(np.int64) for n in ("gate", "up")}
    most = int(550 / np.sqrt(hidden))  # so that a sum stays below 2^12, four and a half deviations out
    x = rng.integers(-most, most + 1, size=(tokens, hidden))
    h = (x @ w["gate"].T) * (x @ w["up"].T)
    assert np.abs(h).max() < 2 ** 24 and (cut(h, 2) != h).any() and np.array_equal(cut(h, 3), h)
    column = rng.integers(0, inter, size=hidden)
    column[:4] = np.argsort(-np.abs(cut(h, 2) - h).max(axis=0))[:4]  # what the last term matters to is among them
    sign = rng.choice([1, -1], size=hidden)
    codes["down"][np.arange(hidden), column] = np.where(sign > 0, ONE, ONE | MINUS)
    scales["gate"][:], scales["up"][:] = 127 + exponent // 2, 127 + exponent - exponent // 2
    got = run(gpu, x.astype(np.float32), codes, scales, hidden, inter)
    assert np.array_equal(got.astype(np.float64), np.ldexp((h[:, column] * sign).astype(np.float64), exponent))
