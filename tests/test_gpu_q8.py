"""The 8-bit cache's operators on the GPU against their plain restatement (oracle/q8.py, float64).

Codes, exponents, read-back values and 32-bit rotations are compared bit for bit. Attention is compared element by
element with a bound that follows from its arithmetic: a score is a sum of 128 products, q carried to 2^-22 of the row's
largest element, summed in 32 bits (each of the 128 additions within 2^-23 of the partial sum, the tensor cores may
truncate); ex2 is good to 2^-22 relative and to the 2^-23 rounding of its argument, which is below 2^7 here; weights are
carried to 2^-21 (f16 pairs) or 2^-11 (one f16: 16-bit prompts); the sums over n tokens add n * 2^-23. Everything is
relative to sum p |v|, and the output adds half an ulp (2^-8 of the value at most in 16 bits, 2^-24 in 32).
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import q8 as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def al():
    import attention_lab_b200
    return attention_lab_b200


def status():
    from attention_lab_b200 import _lib
    return _lib.device_status()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def features(g, *shape):
    x = torch.randn(*shape, generator=g) * torch.exp(torch.randn(*shape[:-1], 1, generator=g))
    return x * torch.where(torch.rand(shape[-1], generator=g) < 0.05, 8.0, 1.0)


def host(x):
    return x.detach().float().cpu().numpy() if x.dtype != torch.float8_e4m3fn else x.view(torch.uint8).cpu().numpy()


def random_cache(seed, B, G, C, spread=0):
    """A cache of random codes and exponents, NaN codes nowhere; `spread` varies the exponents from block to block."""
    g = gen(seed)
    nb = -(-C // 64)
    parts = []
    for _ in range(2):
        c = ref.encode((torch.randn(B, G, C, 128, generator=g) * 60).clamp(-440, 440).numpy())
        parts.append(torch.from_numpy(c).to(DEV).view(torch.float8_e4m3fn))
    exps = [(-6 + torch.randint(-spread, spread + 1, (B, G, nb), generator=g)).to(torch.int8).to(DEV) for _ in range(2)]
    return al().Q8Cache(parts[0], parts[1], exps[0], exps[1])


# ---------------------------------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d, rot", [(128, 128), (128, 96), (128, 64), (128, 20), (128, 2), (64, 64), (8, 6), (200, 144)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotary_matches_bit_for_bit(layout, d, rot, dtype):
    g = gen(d * rot)
    B, H, G, T = 2, 5, 3, 37
    table = al().rotary_table(400, rot, base=1e4, scaling={"type": "yarn", "factor": 4, "original": 100}, device=DEV)
    q = torch.randn(B, T, H, d, generator=g).to(TYPES[dtype]).to(DEV).transpose(1, 2)       # strided, as a layer has it
    k = torch.randn(B, T, G, d, generator=g).to(TYPES[dtype]).to(DEV).transpose(1, 2)
    pos = torch.randint(0, 400, (B, T), generator=g)
    pos[0, :5] = -1
    for inverse in (False, True):
        qo, ko = al().rotary_embed(q, k, table, pos.to(DEV), layout=layout, inverse=inverse)
        for x, y in ((q, qo), (k, ko)):
            assert y.is_contiguous() and y.dtype == x.dtype
            want = ref.rotate(host(x), host(table), pos.numpy()[:, None], layout, inverse)
            want = torch.from_numpy(want).to(TYPES[dtype]).float().numpy()
            assert np.array_equal(host(y), want)
    only, none = al().rotary_embed(q, None, table, 11, layout=layout)
    assert none is None
    both, _ = al().rotary_embed(q, k, table, torch.arange(11, 11 + T, device=DEV), layout=layout)
    assert torch.equal(only, both) and status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(layout):
    """The inverse rotation is the gradient: against central differences (the map is linear, so a step of 1 has no
    truncation error; each side is good to 2^-22 of the loss) and against the transpose of the formula."""
    g = gen(3)
    table = al().rotary_table(64, 32, device=DEV, scaling={"type": "yarn", "factor": 2, "original": 16})
    x = torch.randn(1, 1, 4, 128, generator=g).to(DEV)
    w = torch.randn(1, 1, 4, 128, generator=g).to(DEV)
    grad, _ = al().rotary_embed(w, None, table, 20, layout=layout, inverse=True)
    probe = torch.eye(512, device=DEV).view(512, 1, 4, 128)
    up, _ = al().rotary_embed(x + probe, None, table, 20, layout=layout)
    down, _ = al().rotary_embed(x - probe, None, table, 20, layout=layout)
    diff = ((up.double() - down.double()) * w.double()).sum(dim=(1, 2, 3)) / 2
    assert float((diff - grad.double().view(-1)).abs().max()) < 64 * 2 ** -23
    want = ref.rotate(host(w).astype(np.float64), host(table).astype(np.float64), np.arange(20, 24), layout, True)
    assert np.abs(host(grad) - want).max() < 8 * 2 ** -23


def test_rotary_edges():
    table = al().rotary_table(10, 128, device=DEV)
    q = torch.randn(1, 2, 3, 128, device=DEV)
    out, _ = al().rotary_embed(q, None, table, torch.tensor([[8, 9, 10]], device=DEV))
    assert status() == 4 and torch.all(out[:, :, 2] == 0) and torch.all(out[:, :, 1] != 0)
    assert al().rotary_embed(q[:, :, :0], None, table, 0)[0].shape == (1, 2, 0, 128)
    odd = torch.randn(1, 2, 3, 133, device=DEV)[..., 5:]                      # rows off a 16-byte boundary
    assert torch.equal(al().rotary_embed(odd, None, table, 2)[0], al().rotary_embed(odd.contiguous(), None, table, 2)[0])
    for bad in (lambda: al().rotary_embed(q, None, table, 8), lambda: al().rotary_embed(q, None, table, 0, layout="x"),
                lambda: al().rotary_embed(q, None, table.double(), 0), lambda: al().rotary_embed(q.half(), None, table, 0),
                lambda: al().rotary_embed(q, q[:, :, :2], table, 0),
                lambda: al().rotary_embed(q, None, torch.zeros(10, 130, device=DEV), 0),
                lambda: al().rotary_embed(q, None, table, torch.zeros(1, 3, dtype=torch.int32, device=DEV)),
                lambda: al().rotary_embed(q[..., :4], None, table, 0)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------------------------------------------------
# the quantising write and the read-back
# ---------------------------------------------------------------------------------------------------------------------
def ref_append(cache, k_new, v_new, lengths, table=None, layout="half"):
    """The restatement applied to a host copy of the cache; returns (k, v, k_exp, v_exp)."""
    parts = [host(cache.k).copy(), host(cache.v).copy(), cache.k_exp.cpu().numpy().copy(), cache.v_exp.cpu().numpy().copy()]
    T = k_new.shape[2]
    for b, n in enumerate(lengths):
        k = host(k_new)[b]
        if table is not None:
            k = ref.rotate(k, host(table), np.arange(n - T, n), layout)
        for g in range(k.shape[0]):
            ref.append(parts[0][b, g], parts[2][b, g], k[g], n)
            ref.append(parts[1][b, g], parts[3][b, g], host(v_new)[b, g], n)
    return parts


def same_cache(cache, want):
    for name, x, y in zip(("k", "v", "k_exp", "v_exp"), cache, want):
        x = x.view(torch.uint8).cpu().numpy() if x.dtype == torch.float8_e4m3fn else x.cpu().numpy()
        if x.dtype == np.uint8:                       # both NaN codes are NaN
            x, y = np.where((x & 127) == 127, 127, x), np.where((y & 127) == 127, 127, y)
        assert np.array_equal(x, y), f"{name}: {int((x != y).sum())} differ"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T, lengths", [(1, [1, 64, 65, 200]), (2, [2, 65, 64, 199]), (63, [63, 64, 127, 200]),
                                        (64, [64, 100, 128, 1]), (65, [65, 200, 30, 0]), (200, [200, 5, 64, 129])])
@pytest.mark.parametrize("rot", [0, 128, 20])
def test_append_matches_bit_for_bit(dtype, T, lengths, rot):
    """Every written row and every exponent, rows and blocks that are not written untouched, padding rows dropped."""
    g = gen(T + rot)
    B, G, h, C = 4, 3, 2, 200
    cache = random_cache(5, B, G, C, spread=3)
    k = features(g, B, T, G, 128).to(TYPES[dtype]).to(DEV).transpose(1, 2)
    v = features(g, B, T, G, 128).to(TYPES[dtype]).to(DEV).transpose(1, 2)
    q = torch.randn(B, T, G, h, 128, generator=g).to(TYPES[dtype]).to(DEV).permute(0, 2, 3, 1, 4) if rot else None
    table = al().rotary_table(C, rot, device=DEV) if rot else None
    want = ref_append(cache, k, v, lengths, table)
    got = al().append_q8(cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), k, v, q=q, table=table)
    same_cache(cache, want)
    if rot:
        pos = np.stack([np.arange(n - T, n) for n in lengths])[:, None, None]
        wq = torch.from_numpy(ref.rotate(host(q), host(table), pos, "half")).to(TYPES[dtype]).float().numpy()
        assert np.array_equal(host(got), wq)
    else:
        assert got is None
    assert status() == 0


def test_append_token_by_token_and_growing_blocks():
    """A block written in pieces, each louder than the last: the kept codes are rounded again at every growth."""
    g = gen(8)
    B, G, C = 1, 2, 130
    cache = al().Q8Cache.empty(B, G, C, DEV)
    cache.k.view(torch.uint8).zero_(), cache.v.view(torch.uint8).zero_()
    n = 0
    for step, T in enumerate([1, 1, 1, 30, 1, 40, 1, 55]):
        k = features(g, B, G, T, 128).to(DEV) * 3.0 ** step * 1e-3
        v = features(g, B, G, T, 128).to(DEV) * 0.2 ** step
        n += T
        want = ref_append(cache, k, v, [n])
        al().append_q8(cache, n, k, v)
        same_cache(cache, want)


def test_append_special_values():
    C = 192
    cache = al().Q8Cache.empty(1, 1, C, DEV)
    k = torch.zeros(1, 1, C, 128)
    k[0, 0, 3, 5], k[0, 0, 4, 6], k[0, 0, 5, 7], k[0, 0, 6, 8] = math.nan, math.inf, -math.inf, -0.0
    k[0, 0, 64] = 3.3e38                               # the top of the range
    k[0, 0, 70] = 1e30
    k[0, 0, 130] = 1e-35                               # under the lowest exponent's smallest code
    v = torch.full((1, 1, C, 128), -1e-38)
    want = ref_append(cache, k, v, [C])
    al().append_q8(cache, C, k.to(DEV), v.to(DEV))
    same_cache(cache, want)
    assert cache.k_exp.view(-1).tolist() == [-100, 120, -100]
    kk, _ = al().read_q8(cache, 0, 64, dtype=torch.float32)
    bad = torch.isnan(kk[0, 0]).nonzero().tolist()
    assert bad == [[3, 5], [4, 6], [5, 7]] and torch.isfinite(kk[0, 0, 0]).all()


def test_append_lengths_past_the_capacity_and_stale_blocks():
    g = gen(2)
    cache = random_cache(1, 2, 2, 100)
    k = features(g, 2, 2, 10, 128).to(DEV)
    want = ref_append(cache, k, k, [105, 100])
    al().append_q8(cache, torch.tensor([105, 100], dtype=torch.int32, device=DEV), k, k)
    same_cache(cache, want)
    assert status() == 4
    before = [x.clone() for x in cache]
    al().append_q8(cache, torch.tensor([-7, 2 ** 31 - 1], dtype=torch.int32, device=DEV), k, k)
    assert status() == 4
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    # a block that starts over takes its own exponent, not the one an earlier use left
    cache.k_exp.fill_(50)
    al().append_q8(cache, 10, k, k)
    assert int(cache.k_exp.max()) == 50 and int(cache.k_exp[..., 0].max()) < 10


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lo, hi", [(0, 515), (61, 66), (514, 515), (64, 128), (3, 3)])
def test_read_back(dtype, lo, hi):
    cache = random_cache(4, 2, 3, 515, spread=20)
    k, v = al().read_q8(cache, lo, hi, dtype=TYPES[dtype])
    for got, codes, exps in ((k, cache.k, cache.k_exp), (v, cache.v, cache.v_exp)):
        want = ref.values(host(codes), exps.cpu().numpy())[:, :, lo:hi]
        want = torch.from_numpy(want).float().to(TYPES[dtype])
        assert got.shape == want.shape and torch.equal(got.cpu(), want)


def test_cache_refusals():
    c = al().Q8Cache.empty(2, 2, 100, DEV)
    x = torch.randn(2, 2, 5, 128, device=DEV)
    t = al().rotary_table(100, device=DEV)
    q = torch.randn(2, 2, 3, 5, 128, device=DEV)
    for bad in (lambda: al().append_q8(c, 4, x, x), lambda: al().append_q8(c, 101, x, x),
                lambda: al().append_q8(c, 5, x, x[:, :, :4]), lambda: al().append_q8(c, 5, x, x.bfloat16()),
                lambda: al().append_q8(c, 5, x, x, q=q), lambda: al().append_q8(c, 50, x, x, table=t[:40].contiguous()),
                lambda: al().append_q8(c, 5, x[..., :64], x[..., :64]), lambda: al().append_q8(c, 5, x.half(), x.half()),
                lambda: al().append_q8(c._replace(k=c.k.view(torch.uint8)), 5, x, x),
                lambda: al().append_q8(c._replace(v_exp=c.v_exp[..., :1]), 5, x, x),
                lambda: al().append_q8(c, torch.tensor([5, 5], device=DEV), x, x),
                lambda: al().append_q8(c, 5, x, x, q=q[:, :, :, :4], table=t),
                lambda: al().read_q8(c, -1, 5), lambda: al().read_q8(c, 6, 5), lambda: al().read_q8(c, 0, 101),
                lambda: al().read_q8(c, 0, 5, dtype=torch.float16),
                lambda: al().attend_q8(q, c, 101), lambda: al().attend_q8(q, c, -1),
                lambda: al().attend_q8(q, c, 50, window=-1), lambda: al().attend_q8(q, c, 50, sinks=-1),
                lambda: al().attend_q8(q[..., :64], c, 50), lambda: al().attend_q8(q.half(), c, 50),
                lambda: al().attend_q8(q, c, 50, scale=math.nan), lambda: al().attend_q8(q[:1], c, 50)):
        with pytest.raises(ValueError):
            bad()
    assert al().attend_q8(q[:, :, :, :0], c, 50).shape == (2, 2, 3, 0, 128)
    empty = al().Q8Cache.empty(0, 2, 100, DEV)
    assert al().attend_q8(q[:0], empty, 50).shape == (0, 2, 3, 5, 128)


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def check_attend(cache, q, lengths, window, sinks, out, scale=None):
    k, v = ref.values(host(cache.k), cache.k_exp.cpu().numpy()), ref.values(host(cache.v), cache.v_exp.cpu().numpy())
    B, G, h, T, d = q.shape
    scale = 1 / math.sqrt(d) if scale is None else scale
    x, got = host(q).astype(np.float64), host(out).astype(np.float64)
    one_term = q.dtype == torch.bfloat16 and h * T > 16                  # 16-bit prompts: weights in one f16
    for b in range(B):
        for g in range(G):
            n = int(lengths[b])
            want, mass, mag = ref.attend(x[b, g], k[b, g], v[b, g], n, window, sinks, scale)
            ds = (128 * 2 ** -23 + 2 ** -22) * mag + 2 ** 7 * 2 ** -23      # a score's error (natural log), argument rounding
            rel = 2 * (ds + 2 ** -21 + (2 ** -11 if one_term else 0.0) + n * 2 ** -23)
            tol = rel * mass + (2 ** -8 if q.dtype == torch.bfloat16 else 2 ** -24) * np.abs(want)
            err = np.abs(got[b, g] - want)
            assert np.all(err <= tol), f"b {b} g {g}: error {err.max():.3g}, {float((err / np.maximum(tol, 1e-300)).max()):.3g} of its bound"


def make_q(seed, B, G, h, T, dtype):
    return torch.randn(B, T, G, h, 128, generator=gen(seed)).to(TYPES[dtype]).to(DEV).permute(0, 2, 3, 1, 4)


SHAPES = [(1, 1), (4, 1), (8, 1), (3, 2), (9, 1), (16, 1), (5, 3),       # few columns
          (17, 1), (1, 40), (4, 70), (3, 130), (1, 150), (17, 9), (64, 3)]  # short chunks, prompts


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", SHAPES)
def test_attend_lengths(dtype, h, T):
    lengths = [0, 1, 63, 64, 65, 200, 333]
    cache = random_cache(h + T, len(lengths), 2, 333, spread=2)
    q = make_q(T, len(lengths), 2, h, T, dtype)
    out = al().attend_q8(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    check_attend(cache, q, lengths, 0, 0, out)
    assert torch.all(out[0] == 0) and status() == 0
    one = al().attend_q8(q, cache, 200)
    check_attend(cache, q, [200] * len(lengths), 0, 0, one)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(4, 1), (2, 4), (2, 100), (4, 300)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (64, 4), (100, 64), (129, 200), (1000, 4), (33, 1000), (128, 0)])
def test_attend_window_and_sinks(dtype, h, T, window, sinks):
    lengths = [700, 450, 130, 3]
    cache = random_cache(window + sinks, 4, 1, 700, spread=1)
    q = make_q(window, 4, 1, h, T, dtype)
    out = al().attend_q8(q, cache, torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window, sinks=sinks)
    check_attend(cache, q, lengths, window, sinks, out)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 30, 90])
def test_attend_long_context_split(dtype, T):
    """One request: the key range is split over CTAs and merged."""
    n = 9000
    cache = random_cache(T, 1, 1, n + 5, spread=2)
    q = make_q(7, 1, 1, 2, T, dtype)
    for L in (n, 4097, 70):
        check_attend(cache, q, [L], 0, 0, al().attend_q8(q, cache, torch.tensor([L], dtype=torch.int32, device=DEV)))
        # what the caller knows of the length chooses another split, not another result
        check_attend(cache, q, [L], 0, 0, al().attend_q8(q, cache, torch.tensor([L], dtype=torch.int32, device=DEV),
                                                          max_length=L))
        check_attend(cache, q, [L], 500, 4, al().attend_q8(q, cache, L, window=500, sinks=4))


@pytest.mark.parametrize("h, T", [(2, 1), (1, 7), (2, 40)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (1000, 33), (1023, 1), (8000, 95)])
def test_attend_split_covers_every_token(h, T, window, sinks):
    """Splits by runs of tokens: windows and sinks that straddle a step more at either end, lengths far below and above
    what the caller says (a hint that is too small must not lose tokens)."""
    C = 20011
    cache = random_cache(h, 2, 1, C, spread=1)
    q = make_q(T, 2, 1, h, T, "f32")
    for lengths in ([C, 513], [8191, 16385]):
        on_gpu = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        for hint in (None, C, 3000, 1):
            out = al().attend_q8(q, cache, on_gpu, window=window, sinks=sinks, max_length=hint)
            check_attend(cache, q, lengths, window, sinks, out)
    assert status() == 0


@pytest.mark.parametrize("h, T", [(4, 1), (3, 2), (4, 60)])
def test_attend_scales(h, T):
    """Exponents far apart from block to block (a quiet block may carry all the weight), large and tiny q, negative
    and zero softmax scale."""
    cache = random_cache(3, 2, 1, 400, spread=0)
    q = make_q(4, 2, 1, h, T, "f32")
    cache.v_exp.copy_(torch.tensor([-40, 20, -6, 0, 60, -90, -30], dtype=torch.int8).expand(2, 1, 7))
    check_attend(cache, q, [400, 390], 0, 0, al().attend_q8(q, cache, torch.tensor([400, 390], dtype=torch.int32, device=DEV)))
    cache.k_exp.copy_(torch.tensor([-30, -6, -8, -100, -5, -7, -9], dtype=torch.int8).expand(2, 1, 7))
    for scale in (None, -0.05, 1e-3, 0.0):
        check_attend(cache, q, [400, 400], 0, 0, al().attend_q8(q, cache, 400, scale=scale), scale)
    for size in (1e-20, 1e-3, 30.0):
        check_attend(cache, q * size, [400, 400], 0, 0, al().attend_q8(q * size, cache, 400, scale=0.02), 0.02)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(4, 1), (2, 4), (2, 100)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (90, 4)])
def test_attend_nan_only_where_it_is_seen(dtype, h, T, window, sinks):
    """NaN codes in rows a query does not see never reach it (stale slots, rows before the window, later rows of the
    chunk); where it does see one, K makes the whole row NaN and V its dimension."""
    n, C = 420, 500
    q = make_q(6, 1, 1, h, T, dtype)
    clean = random_cache(9, 1, 1, C)
    base = al().attend_q8(q, clean, n, window=window, sinks=sinks)
    hidden = clean._replace(k=clean.k.clone(), v=clean.v.clone())
    gone = list(range(n, C))
    if window:
        gone += list(range(sinks, n - T - window + 1))
    for x in (hidden.k, hidden.v):
        x.view(torch.uint8)[:, :, gone] = 0x7F
    assert torch.equal(al().attend_q8(q, hidden, n, window=window, sinks=sinks), base)
    # a row that only the chunk's last query sees, and one that all see
    for j, dim in ((n - 1, 17), (n - T, 90)):
        for which in ("k", "v"):
            c = clean._replace(k=clean.k.clone(), v=clean.v.clone())
            getattr(c, which).view(torch.uint8)[0, 0, j, dim] = 0xFF
            got = al().attend_q8(q, c, n, window=window, sinks=sinks)[0, 0]
            for t in range(T):
                row, want = got[:, t], base[0, 0, :, t]
                if not ref.sees(n - T + t, np.array(j), window, sinks):
                    assert torch.equal(row, want)
                elif which == "k":
                    assert torch.isnan(row).all()
                else:
                    assert torch.isnan(row[:, dim]).all()
                    keep = [i for i in range(128) if i != dim]
                    assert torch.equal(row[:, keep], want[:, keep])


def test_attend_many_nan_rows():
    """More NaN rows than the prompt kernel lists."""
    cache = random_cache(1, 1, 1, 600)
    q = make_q(1, 1, 1, 2, 200, "bf16")
    base = al().attend_q8(q, cache, 600)
    cache.v.view(torch.uint8)[0, 0, 450:, 3] = 0x7F
    got = al().attend_q8(q, cache, 600)
    seen = torch.arange(400, 600, device=DEV) >= 450
    assert torch.isnan(got[0, 0, :, seen, 3]).all()
    assert torch.equal(got[0, 0, :, ~seen], base[0, 0, :, ~seen])
    keep = [i for i in range(128) if i != 3]
    assert torch.equal(got[..., keep], base[..., keep])


@pytest.mark.parametrize("T", [1, 20, 80])
def test_attend_past_32_bit_offsets(T):
    """A cache of more than 2^32 bytes: the last tokens of the last head."""
    C = (1 << 25) // 2 + 333
    cache = al().Q8Cache.empty(1, 2, C, DEV)
    small = random_cache(2, 1, 2, 320)
    off = (C - 320) // 64 * 64
    for dst, src in zip((cache.k, cache.v), (small.k, small.v)):
        dst.view(torch.uint8)[:, :, off:off + 320] = src.view(torch.uint8)
    cache.k_exp[..., off // 64:off // 64 + 5] = small.k_exp
    cache.v_exp[..., off // 64:off // 64 + 5] = small.v_exp
    assert cache.k.numel() > 1 << 32
    q = make_q(3, 1, 2, 2, T, "f32")
    got = al().attend_q8(q, cache, off + 320, window=230)
    check_attend(small, q, [320], 230, 0, got)
    k, _ = al().read_q8(cache, off, off + 320, dtype=torch.float32)
    assert torch.equal(k, al().read_q8(small, 0, 320, dtype=torch.float32)[0])
    x = torch.randn(1, 2, 3, 128, device=DEV)
    want = ref_append(small, x, x, [320])
    al().append_q8(cache, off + 320, x, x)
    assert np.array_equal(host(cache.k[:, :, off + 256:off + 320]), want[0][:, :, 256:])


@pytest.mark.parametrize("h, T", [(4, 1), (4, 50)])
def test_streams_and_graphs(h, T):
    """On a stream of its own and replayed from a CUDA graph with the lengths changed on the device in between."""
    cache = random_cache(5, 3, 2, 300)
    q = make_q(2, 3, 2, h, T, "bf16")
    lengths = torch.tensor([300, 211, 64], dtype=torch.int32, device=DEV)
    want = al().attend_q8(q, cache, lengths)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = al().attend_q8(q, cache, lengths)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = al().attend_q8(q, cache, lengths)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    lengths.copy_(torch.tensor([120, 300, 299], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, al().attend_q8(q, cache, lengths)) and status() == 0


def test_attend_repeats_bit_for_bit_and_flags_bad_lengths():
    cache = random_cache(5, 2, 2, 3000)
    for h, T in ((4, 1), (4, 40)):
        q = make_q(2, 2, 2, h, T, "f32")
        a, b = al().attend_q8(q, cache, 3000), al().attend_q8(q, cache, 3000)
        assert torch.equal(a, b) and status() == 0
        c = al().attend_q8(q, cache, torch.tensor([3005, -2], dtype=torch.int32, device=DEV))
        assert status() == 4 and torch.all(c[1] == 0)
        check_attend(cache, q, [3000, 0], 0, 0, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts_alone_and_back_to_back(dtype):
    """Short ragged prompts split over the keys, two query tiles a CTA, launched many times alone and back to back: the
    same bits every time and no wait that gives up (late warps must find every barrier's phase)."""
    cache = random_cache(11, 5, 2, 700)
    q = make_q(5, 5, 2, 3, 333, dtype)
    lengths = [641, 201, 311, 531, 421]
    on_gpu = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = al().attend_q8(q, cache, on_gpu)
    assert status() == 0
    check_attend(cache, q[:2], lengths, 0, 0, want[:2])
    for alone in (True, False):
        for _ in range(60):
            got = al().attend_q8(q, cache, on_gpu)
            if alone:
                torch.cuda.synchronize()
                assert status() == 0
        assert torch.equal(got, want) and status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,G,h,T,C,window,lengths", [
    (5, 2, 3, 333, 700, 0, [641, 201, 311, 531, 421]),     # CTAs of 128 rows, some of padding alone
    (3, 4, 5, 200, 1500, 0, [37, 1500, 0]),
    (2, 2, 1, 300, 900, 100, [900, 129]),
    (1, 8, 4, 64, 2048, 0, [2048]),                        # CTAs of 128 rows, keys split
    (2, 4, 2, 130, 1000, 0, [5, 1000]),
    (1, 4, 4, 256, 3000, 0, [2987]),                       # CTAs of 256 rows, keys split
    (1, 1, 8, 520, 3000, 0, [701])])
def test_prompts_of_few_rows(dtype, B, G, h, T, C, window, lengths):
    """Every way a prompt over few rows is spread over the GPU, into memory that held NaN, with rows of padding: each row
    is written once, by the CTA that owns it."""
    cache = random_cache(23, B, G, C)
    q = make_q(24, B, G, h, T, dtype)
    on_gpu = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = None
    for _ in range(20):
        junk = torch.full((B, G, h, T, 128), float("nan"), device=DEV, dtype=q.dtype)
        del junk
        got = al().attend_q8(q, cache, on_gpu, window=window)
        want = got.clone() if want is None else want
        assert torch.equal(got, want) and status() == 0
    check_attend(cache, q, lengths, window, 0, want)


def test_fp32_prompts_do_not_drift():
    """The tensor cores cut sums off towards zero; over a long context that must not add up. With every value one the output
    is one: O loses at most 2^-23 of itself in each of the 32 sums between two additions to the fp32 sum, and the errors of
    those additions and of the denominator, rounded to nearest, average out over the rows."""
    n = 12000
    cache = random_cache(31, 2, 8, n)
    cache.v.copy_(torch.full((2, 8, n, 128), 256.0, device=DEV).to(torch.float8_e4m3fn))
    cache.v_exp.fill_(-8)
    q = make_q(32, 2, 8, 8, 80, "f32")
    out = al().attend_q8(q, cache, torch.tensor([n, n - 77], dtype=torch.int32, device=DEV))
    drift = float((out.double() - 1).mean())
    assert abs(drift) <= 32 * 2 ** -23, drift
    assert status() == 0


def test_misaligned_queries_are_copied():
    cache = random_cache(5, 1, 2, 100)
    wide = torch.randn(1, 2, 3, 1, 131, device=DEV)
    assert torch.equal(al().attend_q8(wide[..., 3:], cache, 90), al().attend_q8(wide[..., 3:].contiguous(), cache, 90))
