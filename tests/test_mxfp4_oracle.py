"""CPU: the tests' own MXFP4 forms, on values worked out by hand, and the plain
forms of perf/more_operators.py against them."""
import os
import sys

import numpy as np
import torch

import mxfp4_oracle as MO

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf"))


def row(*v):
    return np.array(list(v) + [0.0] * (32 - len(v)))[None]


def kept(x):
    return MO.values(*MO.quantize(x))


def test_codes_and_scales():
    qs, s = MO.quantize(row(4.0, -6.0, 0.5, -1.5))
    assert s.tolist() == [[127]] and qs[0, :2].tolist() == [0xF6, 0xB1]
    assert MO.quantize(row())[1].tolist() == [[0]]
    assert MO.quantize(row(2.0**-130))[1].tolist() == [[0]]  # below the smallest scale's reach
    assert MO.quantize(row(2.0**127))[1].tolist() == [[252]]
    assert MO.quantize(row(np.inf))[1].tolist() == [[255]] and MO.quantize(row(1.0, np.nan))[1].tolist() == [[255]]
    assert np.isnan(MO.values(*MO.quantize(row(np.nan)))).all()


def test_ties_go_to_even_and_past_six_is_six():
    x = row(4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.25, -0.75, -5.0, 0.2500001, 0.7499999)
    assert kept(x)[0, :14].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, -0.0, -1, -4, 0.5, 0.5]


def test_every_code_comes_back():
    g = np.concatenate((MO.GRID, -MO.GRID))
    for e in (-127, -20, 0, 100):
        x = np.ldexp(np.concatenate((g, g))[None], e)
        qs, s = MO.quantize(x)
        assert s[0, 0] == 127 + e and np.array_equal(MO.values(qs, s), x)


def test_plain_forms_of_the_measured_cases():
    import more_operators as mo
    r = np.random.default_rng(3)
    x = (r.standard_normal((40, 96)) * np.exp(3 * r.standard_normal((40, 1)))).astype(np.float32)
    x[3] = 0
    x[5, :32] = 1e-39
    qs, s = mo._quantized(torch.from_numpy(x))
    wq, ws = MO.quantize(x.astype(np.float64))
    assert np.array_equal(qs.numpy(), wq) and np.array_equal(s.numpy(), ws)
    assert np.array_equal(mo._values(qs, s).double().numpy(), MO.values(wq, ws))
