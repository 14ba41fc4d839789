"""The fit behind the erf form of gelu and the series behind the rotation, from the constants in the sources."""
import math
import os
import re

import numpy as np

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ltx-2.5-swift_b200", "csrc")


def source(name):
    return open(os.path.join(CSRC, name)).read()


def erf_fit():
    """(slope of the argument, coefficients from the highest power down) in activate's last branch."""
    text = source("ffn_common.cuh")
    text = text[text.index("// erfc(x / sqrt 2) / 2 ="):]
    text = text[:text.index("const float s = g < 0.0f")]
    scale = float(re.search(r"fmaf\(([\d.]+)f, x, 1\.0f\)", text).group(1))
    first, second = re.search(r"float q = fmaf\(t, (-?[\d.e-]+)f, (-?[\d.e-]+)f\)", text).groups()
    rest = re.findall(r"q = fmaf\(t, q, (-?[\d.e-]+)f\)", text)
    coefficients = [float(first), float(second)] + [float(c) for c in rest if c]
    assert len(coefficients) == 8
    return scale, coefficients


def scaled_erfc(x):
    """e^(x^2 / 2) erfc(x / sqrt 2) / 2 by its continued fraction where erfc itself has too few digits left."""
    if x < 5:
        return math.exp(0.5 * x * x) * math.erfc(x / math.sqrt(2)) / 2
    f = 0.0
    for n in range(200, 0, -1):  # erfc's Laplace fraction: 1 / (x + 1 / (x + 2 / (x + ...)))
        f = n / (x + f)
    return 1 / (x + f) / math.sqrt(2 * math.pi)


def test_the_fit_is_within_what_its_comment_says():
    scale, coefficients = erf_fit()
    worst = 0.0
    for x in np.linspace(0, 14, 20001):
        t = 1 / (1 + scale * x)
        q = 0.0
        for c in coefficients:
            q = q * t + float(np.float32(c))
        worst = max(worst, abs(q / scaled_erfc(x) - 1))
    assert 3.7e-7 < worst <= 3.8e-7, worst


def test_the_continued_fraction_meets_erfc():
    for x in (2.0, 5.0, 8.0):
        direct = math.exp(0.5 * x * x) * math.erfc(x / math.sqrt(2)) / 2
        f = 0.0
        for n in range(200, 0, -1):
            f = n / (x + f)
        assert abs(1 / (x + f) / math.sqrt(2 * math.pi) / direct - 1) < 1e-12


def test_the_series_of_the_rotation_is_within_what_its_comment_says():
    text = source("rotary_embed.cu")
    text = text[text.index("float ps = "):text.index("const int q = __double2loint")]
    assert re.search(r"1\.0f / 362880, -1\.0f / 5040", text) and re.search(r"-1\.0f / 3628800, 1\.0f / 40320", text)
    sine = cosine = 0.0
    for x in np.linspace(1e-3, math.pi / 4, 20001):
        s = sum((-1) ** k * x ** (2 * k + 1) / math.factorial(2 * k + 1) for k in range(5))
        c = sum((-1) ** k * x ** (2 * k) / math.factorial(2 * k) for k in range(6))
        sine, cosine = max(sine, abs(s / math.sin(x) - 1)), max(cosine, abs(c / math.cos(x) - 1))
    assert 2.0 ** -28.6 < sine <= 2.0 ** -28.5, math.log2(sine)
    assert cosine <= 2.0 ** -32, math.log2(cosine)
