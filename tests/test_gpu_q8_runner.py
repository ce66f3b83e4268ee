"""The Qwen3 driver over an 8-bit cache (runner.make_state(..., cache_format="q8")): what its attention modules read and
return, layer by layer, against the restatement of the format (oracle/q8.py), on a tiny Qwen3 with the kernels' head
dimension. The bound is that of tests/test_gpu_q8.py."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import q8 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rn():
    from attention_lab_b200 import runner
    return runner


def ids(n, seed=1, vocab=256):
    return torch.randint(0, vocab, (1, n), generator=torch.Generator().manual_seed(seed)).to(DEV)


def host_codes(x):
    return x.view(torch.uint8).cpu().numpy()


def bound(q, n, mass, mag, want, dtype, one_term):
    ds = (128 * 2 ** -23 + 2 ** -22) * mag + 2 ** 7 * 2 ** -23
    rel = 2 * (ds + 2 ** -21 + (2 ** -11 if one_term else 0.0) + n * 2 ** -23)
    return rel * mass + (2 ** -8 if dtype == torch.bfloat16 else 2 ** -24) * np.abs(want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window, sinks", [(0, 0), (50, 4)])
def test_every_layer_reads_its_cache(dtype, window, sinks):
    r = rn()
    with torch.inference_mode():
        m = r.tiny_qwen3(dtype=dtype, device=DEV)
        holder = r.wrap_model(m)
        st = r.make_state(m, 300, "full", cache_format="q8", window=window, sinks=sinks)
        run = r.LabRunner(m, holder, st)
        L = len(m.model.layers)
        cap = [dict() for _ in range(L)]
        for l, layer in enumerate(m.model.layers):
            inner = layer.self_attn.inner
            inner.q_norm.register_forward_hook(lambda mod, i, o, l=l: cap[l].__setitem__("q", o.clone()))
            inner.k_norm.register_forward_hook(lambda mod, i, o, l=l: cap[l].__setitem__("k", o.clone()))
            inner.v_proj.register_forward_hook(lambda mod, i, o, l=l: cap[l].__setitem__("v", o.clone()))
            inner.o_proj.register_forward_pre_hook(lambda mod, i, l=l: cap[l].__setitem__("o", i[0].clone()))
        table = st.cache.table.cpu().numpy()
        prompt = ids(150)
        at = 0
        for n, phase in ((100, "prefill"), (49, "prefill"), (1, "prefill"), (1, "decode"), (1, "decode")):
            before = [[host_codes(x) if x.dtype != torch.int8 else x.cpu().numpy() for x in kv] for kv in st.cache.kv]
            tok = prompt[:, at:at + n] if phase == "prefill" else ids(1, seed=at)
            run.forward(tok, phase=phase)
            pos = np.arange(at, at + n)
            at += n
            for l in range(L):
                G, h = st.cache.groups, m.config.num_attention_heads // st.cache.groups
                k = cap[l]["k"][0].float().cpu().numpy().transpose(1, 0, 2)                       # [G,T,d] before rotation
                v = cap[l]["v"][0].float().cpu().numpy().reshape(n, G, 128).transpose(1, 0, 2)
                q = cap[l]["q"][0].float().cpu().numpy().transpose(1, 0, 2).reshape(G, h, n, 128)
                k = ref.rotate(k, table, pos, "half")
                q = torch.from_numpy(ref.rotate(q, table, pos, "half")).to(dtype).double().numpy()
                kc, vc, ke, ve = before[l]
                for g in range(G):
                    ref.append(kc[0, g], ke[0, g], k[g], at)
                    ref.append(vc[0, g], ve[0, g], v[g], at)
                now = st.cache.kv[l]
                assert np.array_equal(host_codes(now.k)[:, :, :at], kc[:, :, :at])
                assert np.array_equal(host_codes(now.v)[:, :, :at], vc[:, :, :at])
                kk, vv = ref.values(kc, ke), ref.values(vc, ve)
                got = cap[l]["o"][0].double().cpu().numpy().reshape(n, G, h, 128).transpose(1, 2, 0, 3)
                for g in range(G):
                    want, mass, mag = ref.attend(q[g], kk[0, g], vv[0, g], at, window, sinks, 1 / math.sqrt(128))
                    tol = bound(q, at, mass, mag, want, dtype, dtype == torch.bfloat16 and h * n > 16)
                    assert np.all(np.abs(got[g] - want) <= tol), (l, g, at)
        assert st.cache.valid_length == 152


def test_rollback_branch_and_stale_slots():
    r = rn()
    with torch.inference_mode():
        m = r.tiny_qwen3(device=DEV)
        holder = r.wrap_model(m)
        st = r.make_state(m, 256, "full", cache_format="q8")
        run = r.LabRunner(m, holder, st)
        run.prefill(ids(128), 64)
        for kv in st.cache.kv:                               # nothing past the length is ever read
            for x in (kv.k, kv.v):
                x.view(torch.uint8)[:, :, 128:] = 0x7F
        branch = st.cache.clone()
        a = [run.step(ids(1, seed=s)).clone() for s in (5, 6, 7)]
        assert all(torch.isfinite(x).all() for x in a) and st.cache.valid_length == 131
        run.rollback(128)                                    # a block boundary: the same tokens give the same bits
        b = [run.step(ids(1, seed=s)).clone() for s in (5, 6, 7)]
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        st2 = r.LabState(branch, None, mode="full")
        c = [r.LabRunner(m, holder, st2).step(ids(1, seed=s)).clone() for s in (5, 6, 7)]
        assert all(torch.equal(x, y) for x, y in zip(a, c)) and st.cache.valid_length == 131
        with pytest.raises(RuntimeError, match="capacity"):
            run.prefill(ids(200), 200)


def test_close_to_the_plain_cache():
    """8-bit K/V against float32 K/V in the same model: codes carry 4 significant bits, so every K and V entry is within
    2^-4 of its value; through softmax averages and two layers the logits stay within a few percent of their spread
    (a wrong position, head or scale gives errors of the order of the spread itself)."""
    r = rn()
    with torch.inference_mode():
        m = r.tiny_qwen3(device=DEV)
        holder = r.wrap_model(m)
        out = {}
        for fmt in ("plain", "q8"):
            run = r.LabRunner(m, holder, r.make_state(m, 256, "full", cache_format=fmt))
            out[fmt] = [run.prefill(ids(200), 64, keep_logits=True)] + [run.step(ids(1, seed=s)) for s in range(3)]
        for a, b in zip(out["plain"], out["q8"]):
            assert float((a - b).norm() / a.norm()) < 0.1


def test_refusals():
    r = rn()
    m = r.tiny_qwen3(device=DEV)
    for bad in (lambda: r.make_state(m, 64, "sparse", cache_format="q8"), lambda: r.make_state(m, 64, "full", cache_format="x"),
                lambda: r.make_state(m, 64, "full", window=5), lambda: r.make_state(m, 64, "full", cache_format="q8", sinks=-1),
                lambda: r.make_state(m, 64, "full", cache_format="q8", decode_backend="sdpa_fold"),
                lambda: r.make_state(m, 0, "full", cache_format="q8")):
        with pytest.raises(ValueError):
            bad()
    plain, eight = r.make_cache(m, 640, with_index=False, dtype=torch.bfloat16), r.make_q8_cache(m, 640)
    assert 0.5 < eight.bytes()["total_bytes"] / plain.bytes()["total_bytes"] < 0.501
