"""The 8-bit cache's host side without a GPU: rotary tables as checkpoints use them."""
from __future__ import annotations

import math

import pytest
import torch

from attention_lab_b200 import q8

transformers = pytest.importorskip("transformers")


def model_rotary(head_dim, length, base, **rope):
    """The rotary module of a Qwen3 configuration."""
    from transformers.models.qwen3.modeling_qwen3 import Qwen3RotaryEmbedding
    cfg = transformers.Qwen3Config(hidden_size=4 * head_dim, num_attention_heads=4, num_key_value_heads=2,
                                   head_dim=head_dim, max_position_embeddings=length)
    cfg.rope_parameters = dict(rope_theta=base, **rope)
    return Qwen3RotaryEmbedding(cfg)


@pytest.mark.parametrize("base, rot, factor, original, turns", [
    (1e6, 128, 4.0, 32768, {}), (1e4, 64, 8.0, 2048, {}), (1e6, 96, 2.0, 4096, {}), (5e5, 128, 16.0, 8192, {}),
    (1e6, 128, 40.0, 4096, {"fast": 48.0, "slow": 2.0}), (1e4, 128, 4.0, 20, {})])
def test_yarn_is_the_table_checkpoints_use(base, rot, factor, original, turns):
    """Every pair, the ramp's middle among them. transformers computes its frequencies in 32 bits (a power and two
    products: 2^-20 relative is ample), so tables are compared where that moves an angle by less than 1e-4."""
    names = {"fast": "beta_fast", "slow": "beta_slow"}
    theirs = model_rotary(rot, int(factor * original), base, rope_type="yarn", factor=factor,
                          original_max_position_embeddings=original, **{names[k]: v for k, v in turns.items()})
    ours = q8.rotary_table(100, rot, base=base, device="cpu",
                           scaling=dict(type="yarn", factor=factor, original=original, **turns)).double()
    ang = torch.arange(100, dtype=torch.float64)[:, None] * theirs.inv_freq.double()
    amp = theirs.attention_scaling
    assert amp == pytest.approx(0.1 * math.log(factor) + 1)
    assert (ours[:, :rot // 2] - amp * ang.cos()).abs().max() < 2e-4
    assert (ours[:, rot // 2:] - amp * ang.sin()).abs().max() < 2e-4
    freq = torch.atan2(ours[1, rot // 2:], ours[1, :rot // 2])           # of position 1: the frequencies themselves
    assert ((freq - theirs.inv_freq.double()) / theirs.inv_freq.double()).abs()[freq > 1e-3].max() < 1e-3


@pytest.mark.parametrize("bad", [dict(original=0), dict(original=-5), dict(slow=0.0), dict(base=1.0)])
def test_yarn_refuses(bad):
    bad = dict(bad)
    base = bad.pop("base", 1e4)
    with pytest.raises(ValueError):
        q8.rotary_table(8, 16, base=base, scaling={"type": "yarn", "factor": 2, "original": 64, **bad}, device="cpu")


@pytest.mark.parametrize("rope", [dict(rope_type="dynamic", factor=2.0),
                                  dict(rope_type="longrope", factor=4.0, short_factor=[1.0] * 64, long_factor=[2.0] * 64,
                                       original_max_position_embeddings=64)])
def test_frequencies_that_change_with_the_length_are_refused(rope):
    from types import SimpleNamespace
    from attention_lab_b200 import runner
    model = SimpleNamespace(model=SimpleNamespace(rotary_emb=model_rotary(128, 256, 1e6, **rope)))
    with pytest.raises(ValueError, match=rope["rope_type"]):
        runner.model_rotary_table(model, 100)


@pytest.mark.parametrize("rope", [dict(rope_type="default"), dict(rope_type="linear", factor=2.0),
                                  dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64),
                                  dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                       original_max_position_embeddings=64)])
def test_a_models_fixed_frequencies_become_its_table(rope):
    from types import SimpleNamespace
    from attention_lab_b200 import runner
    rot = model_rotary(128, 256, 1e6, **rope)
    table = runner.model_rotary_table(SimpleNamespace(model=SimpleNamespace(rotary_emb=rot)), 100).double()
    ang = torch.arange(100, dtype=torch.float64)[:, None] * rot.inv_freq.double()
    assert (table - torch.cat([ang.cos(), ang.sin()], 1) * rot.attention_scaling).abs().max() < 2 ** -23


def test_importing_the_package_maps_no_native_library():
    """Host-side users of the package (selection rules, tables, a CPU measurement) do not load the CUDA library; the first
    operator does."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import torch
import attention_lab_b200 as al
from attention_lab_b200 import q8, runner, selection
al.rotary_table(8, 128, device="cpu"), al.Q8Cache.empty(1, 1, 8, "cpu")
maps = lambda: [l for l in open("/proc/self/maps") if "attention_lab_b200" in l and ".so" in l]
assert not maps(), maps()[:2]
x = torch.zeros(1, 1, 3, 128)
try:
    al.rotary_embed(x, None, torch.zeros(8, 128), 0)
except ValueError as e:
    assert "CUDA" in str(e)
assert maps()
"""
    res = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def test_a_cluster_that_cannot_be_scheduled_is_halved(tmp_path):
    """The token kernel's launch asks for clusters of up to 16; where the device schedules smaller ones only, the largest of
    those is taken, and a failing question ends the launch with its status."""
    import os
    import subprocess
    from pathlib import Path
    from attention_lab_b200 import build
    src = tmp_path / "clusters.cpp"
    src.write_text('''
#include <cstdio>
#include "al_host.h"
int main() {
  for (int want = 1; want <= 16; want *= 2)
    for (int most = 1; most <= 16; most *= 2) {
      int out = -1, asked = 0;
      const int rc = al::fitting_cluster(want, [&](int cs, bool* ok) { ++asked; *ok = cs <= most; return AL_OK; }, &out);
      if (rc != AL_OK || out != (want < most ? want : most)) return std::printf("%d of %d: %d\\n", want, most, out), 1;
      if (want == 1 && asked) return 2;
    }
  int out = -1;
  return al::fitting_cluster(8, [](int, bool*) { return AL_ECUDA; }, &out) == AL_ECUDA && out == -1 ? 0 : 3;
}
''')
    cuda = Path(os.path.realpath(build.nvcc())).parents[1]
    exe = tmp_path / "clusters"
    subprocess.run(["g++", "-std=c++17", "-I", str(build.SRC), "-I", str(cuda / "include"), str(src), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def test_the_build_notices_what_it_was_built_with(monkeypatch, tmp_path):
    """Built files are stale when a source, the build rules, a compiler line, torch or the Python ABI is another."""
    import os
    from attention_lab_b200 import build
    assert build.PKG / "build.py" in build.sources()
    for name in ("LIB", "BIND", "STAMP"):
        monkeypatch.setattr(build, name, tmp_path / name)
    assert not build.up_to_date()
    build.LIB.touch(), build.BIND.touch()
    assert not build.up_to_date()                                     # nothing says what they were built with
    build.STAMP.write_text(build.stamp())
    assert build.up_to_date()
    with monkeypatch.context() as m:
        m.setattr(build, "ARCH", [*build.ARCH, "-DSOMETHING"])
        assert not build.up_to_date()
    with monkeypatch.context() as m:
        m.setattr(build.importlib.metadata, "version", lambda name: "0.0")
        assert not build.up_to_date()
    with monkeypatch.context() as m:
        m.setattr(build.sysconfig, "get_config_var", lambda name: "other")
        assert not build.up_to_date()
    assert build.up_to_date()
    newest = max(s.stat().st_mtime for s in build.sources())
    os.utime(build.BIND, (newest - 10, newest - 10))
    assert not build.up_to_date()


def test_a_state_over_an_8_bit_cache_refuses_what_it_cannot_use():
    from attention_lab_b200 import runner
    cache = runner.Q8LabCache(layers=2, batch=1, groups=1, capacity=64, head_dim=128, table=torch.zeros(64, 128), device="cpu")
    assert runner.LabState(cache, window=8, sinks=1).eight_bit
    for kw in (dict(sparse_layers=[0]), dict(selector="recent"), dict(selector="uniform"), dict(indexers=[None, None]),
               dict(canonical_order=True)):
        with pytest.raises(ValueError, match="8-bit"):
            runner.LabState(cache, **kw)


def test_the_attention_bound_notices_a_lost_low_term():
    """tests/q8_bounds.py against its own planted mistakes: two-term weights stay within the two-term bound, weights cut to
    one f16 term do not, and the one-term bound holds those."""
    import numpy as np
    import q8_bounds
    from oracle import q8 as ref
    rng = np.random.default_rng(0)
    n = 24
    q = rng.normal(size=(17, 1, 128))
    k = ref._VALUES[ref.encode(np.clip(rng.normal(size=(n, 128)) * 60, -440, 440))] * 2.0 ** -6
    v, e = ref.encode(np.clip(rng.normal(size=(n, 128)) * 60, -440, 440)), np.array([-6], np.int8)

    def one(w):
        return w.astype(np.float16).astype(np.float64)

    def two(w):
        return one(w) + one(w - one(w))

    def run(terms, weight=None, half_ulp=2 ** -8):
        return q8_bounds.attend(q, k, v, e, n, 0, 0, 0.02, terms=terms, out_half_ulp=half_ulp, weight=weight)

    want, tol = run(2)
    assert (np.abs(run(2, two)[0] - want) <= tol).all()
    assert not (np.abs(run(2, one)[0] - want) <= tol).all()
    assert (np.abs(run(1, one)[0] - want) <= run(1)[1]).all()
    # a quiet block under a loud one: two terms end 2^-31 below the row's loudest term, which the bound allows and needs
    e = np.array([-50, 0], np.int8)
    k, v = np.tile(k, (4, 1))[:80], np.tile(v, (4, 1))[:80]
    v[64:, 64:] = 0
    n = 80
    biased = lambda w: two(w * 2.0 ** -4) * 2.0 ** 4
    want, tol = run(2, half_ulp=2 ** -24)
    err = np.abs(run(2, biased, 2 ** -24)[0] - want)
    assert (err <= tol).all() and np.abs(want[..., 64:]).min() > 0 and (err[..., 64:] > 0.5 * np.abs(want[..., 64:])).all()
