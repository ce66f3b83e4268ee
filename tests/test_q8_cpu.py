"""The 8-bit cache without a GPU: the format's restatement against torch's e4m3 type, the rotary table's formulas, and
the operators' refusals."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from attention_lab_b200 import q8
from oracle import q8 as ref


def test_codes_are_torch_e4m3():
    codes = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    got = ref.code_values()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])
    x = torch.cat([torch.linspace(-448, 448, 40001), torch.linspace(-0.02, 0.02, 4001)])
    assert np.array_equal(ref.encode(x.numpy()), x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_exponent_is_the_smallest_that_holds():
    for e in (-100, -17, 0, 5, 120):
        top = math.ldexp(448.0, e)
        assert ref.exponent(top) == e
        if e < 120:
            assert ref.exponent(top * (1 + 2 ** -23)) == e + 1
    assert ref.exponent(0.0) == -100


def test_rotary_table_plain_and_scaled():
    t = q8.rotary_table(50, 16, base=1e4, device="cpu").double().numpy()
    pos, i = np.arange(50)[:, None], np.arange(8)[None]
    ang = pos * 1e4 ** (-2 * i / 16)
    assert np.abs(t[:, :8] - np.cos(ang)).max() < 2 ** -24 and np.abs(t[:, 8:] - np.sin(ang)).max() < 2 ** -24
    lin = q8.rotary_table(50, 16, scaling={"type": "linear", "factor": 4}, device="cpu")
    assert torch.allclose(lin[4 * 7], torch.from_numpy(t[7]).float(), atol=2 ** -24)
    # ntk: the lowest frequency is divided by the factor exactly, the highest is kept
    ntk = q8.rotary_table(50, 16, scaling={"type": "ntk", "factor": 4}, device="cpu").double().numpy()
    low = 1e4 ** (-14 / 16) / 4
    assert np.abs(ntk[:, 8 + 7] - np.sin(np.arange(50) * low)).max() < 1e-7
    assert np.abs(ntk[:, 0] - np.cos(np.arange(50.0))).max() < 1e-7
    yarn = q8.rotary_table(4096, 64, base=1e6, scaling={"type": "yarn", "factor": 4, "original": 1024}, device="cpu")
    amp = 0.1 * math.log(4) + 1
    assert np.abs(yarn[:, 0].double().numpy() - amp * np.cos(np.arange(4096))).max() < 1e-6      # turns often: kept
    low = 1e6 ** (-62 / 64) / 4
    assert np.abs(yarn[:, 63].double().numpy() - amp * np.sin(np.arange(4096) * low)).max() < 1e-6


@pytest.mark.parametrize("bad", [dict(length=0), dict(rotary_dim=7), dict(scaling={"type": "nope", "factor": 2}),
                                 dict(scaling={"type": "yarn", "factor": 2}), dict(scaling={"type": "linear", "factor": 0}),
                                 dict(scaling={"type": "linear", "factor": 2, "extra": 1}),
                                 dict(scaling={"type": "yarn", "factor": 2, "original": 9, "fast": 1, "slow": 2})])
def test_rotary_table_refuses(bad):
    kw = dict(length=8, rotary_dim=8)
    kw.update(bad)
    with pytest.raises(ValueError):
        q8.rotary_table(kw.pop("length"), kw.pop("rotary_dim"), device="cpu", **kw)


def test_operators_refuse_cpu_tensors():
    c = q8.Q8Cache.empty(1, 2, 70, "cpu")
    assert c.k_exp.shape == (1, 2, 2) and c.k.dtype == torch.float8_e4m3fn
    x = torch.zeros(1, 2, 3, 128)
    for call in (lambda: q8.append_q8(c, 3, x, x), lambda: q8.read_q8(c, 0, 3), lambda: q8.attend_q8(x[:, :, None], c, 3),
                 lambda: q8.rotary_embed(x, x, torch.zeros(8, 128), 0)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="capacity"):
        q8.Q8Cache.empty(1, 2, 0, "cpu")
