"""The tanh polynomial of attention's backward pass, from the coefficients in the kernel's source: within the bounds that
stand beside it, with exact arithmetic and in fp32 as the kernel evaluates it."""
import re
from pathlib import Path

import numpy as np

CSRC = Path(__file__).resolve().parent.parent / "pipelink_b200" / "csrc"
NUMBER = r"-?\d+\.\d+(?:e-?\d+)?"


def body(file, name):
    text = (CSRC / file).read_text()
    at = text.index(f"Pair {name}(")
    return text[at:text.index("\n}", at)]


def fma(a, b, c):
    return (a.astype(np.float64) * b.astype(np.float64) + np.float64(c)).astype(np.float32)


def horner(coefficients, u):
    y = np.full_like(u, np.float32(coefficients[0]))
    for c in coefficients[1:]:
        y = fma(y, u, np.float32(c))
    return y


def off_by(t, x):
    return np.log2(np.abs(t.astype(np.float64) / np.tanh(x.astype(np.float64)) - 1).max())


def test_polynomial_of_small_scores():
    text = body("attention_bwd.cu", "tanh_small")
    c = [float(m) for m in re.findall(rf"make_pair\(({NUMBER})f, \1f\)", text)]
    assert len(c) == 5
    end = float(re.search(rf"kSmallCap = ({NUMBER})f", (CSRC / "attention_bwd.cu").read_text()).group(1))
    x = np.linspace(1e-6, end, 2_000_001)
    exact = np.polyval([np.float64(np.float32(v)) for v in c], x * x) * x
    assert np.log2(np.abs(exact / np.tanh(x) - 1).max()) <= -23.35
    x = x.astype(np.float32)
    assert off_by(x * horner(c, x * x), x) <= -22.3
