"""The 8-bit cache's operators on the GPU at their limits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import q8_bounds
from oracle import q8 as ref
from test_gpu_q8 import DEV, TYPES, al, check_attend, gen, host, make_q, random_cache, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(2, 3), (4, 16), (1, 40), (4, 100), (3, 333)])      # single tokens, prompts
def test_a_window_past_the_capacity_hides_nothing(dtype, h, T):
    """Requests padded on the left: positions reach down to -T, and a window that is as large as an int must not wrap
    around below them. Sinks that cover the cache hide nothing either, whatever the window."""
    C, lengths = 350, [350, 5, 1, 0, 100]
    cache = random_cache(h + T, len(lengths), 2, C, spread=1)
    q = make_q(T, len(lengths), 2, h, T, dtype)
    on_gpu = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = al().attend_q8(q, cache, on_gpu)
    check_attend(cache, q, lengths, 0, 0, want)
    for window in (C, C + 1, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1):
        for sinks in (0, 4, 2 ** 31 - 1):
            assert torch.equal(al().attend_q8(q, cache, on_gpu, window=window, sinks=sinks), want), (window, sinks)
    check_attend(cache, q, lengths, 7, 2 ** 31 - 1, al().attend_q8(q, cache, on_gpu, window=7, sinks=2 ** 31 - 1))
    check_attend(cache, q, lengths, C - 1, 3, al().attend_q8(q, cache, on_gpu, window=C - 1, sinks=3))
    assert status() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(1, 1), (4, 2), (1, 60), (2, 90), (1, 300)])
def test_nan_in_a_split_without_weight(dtype, h, T):
    """A visible NaN code in V makes its dimension NaN however far its token's score lies below the row's maximum (0 times
    NaN is NaN), so also where warps, CTAs or key splits that hold it have no weight left; nothing else changes. Every
    score is 0 but the first token's, about 600 binades above."""
    C = 9000
    cache = random_cache(7, 1, 1, C)
    cache.k.view(torch.uint8).zero_()
    cache.k.view(torch.uint8)[0, 0, 0, 0] = 0x7E                       # 448
    cache.k_exp.zero_()
    q = torch.zeros(1, 1, h, T, 128, device=DEV, dtype=TYPES[dtype])
    q[..., 0] = 1.0
    on_gpu = torch.tensor([C], dtype=torch.int32, device=DEV)
    for j in (1, 31, 40, 130, 700, 4100, C - T - 1, C - T):
        bad = cache._replace(v=cache.v.clone())
        bad.v.view(torch.uint8)[0, 0, j, 5] = 0x7F
        for lengths, hint in ((on_gpu, None), (on_gpu, C), (on_gpu, 3000), (on_gpu, 1), (C, None)):
            got = host(al().attend_q8(q, bad, lengths, scale=1.0, max_length=hint))
            base = host(al().attend_q8(q, cache, lengths, scale=1.0, max_length=hint))
            assert np.isnan(got[..., 5]).all(), (j, hint)
            keep = [i for i in range(128) if i != 5]
            assert np.array_equal(got[..., keep], base[..., keep]), (j, hint)
    assert status() == 0


def test_fp32_single_tokens_do_not_drift():
    """As for prompts: with every value one the output is one, and what the tensor cores cut off must not add up over a long
    context that one CTA walks alone (as many segments as SMs, so no split). Between two additions to the fp32 sum a warp
    takes 16 tensor-core sums, each cutting off at most 2^-23 of what it holds; rounded additions average out."""
    B, G, n = 19, 8, 131072
    cache = al().Q8Cache.empty(B, G, n, DEV)
    for b in range(B):
        x = torch.randint(0, 127, (G, n, 128), device=DEV, dtype=torch.uint8, generator=torch.Generator(DEV).manual_seed(b))
        cache.k.view(torch.uint8)[b] = x | (x << 7)                     # any finite code, the lowest bit as its sign
    cache.k_exp.fill_(-14)                                              # scores of the order of one
    cache.v.view(torch.uint8).fill_(0x78)                               # 256
    cache.v_exp.fill_(-8)
    q = make_q(33, B, G, 2, 1, "f32")
    out = al().attend_q8(q, cache, n)
    drift = float((out.double() - 1).mean())
    assert abs(drift) <= 16 * 2 ** -23, drift
    assert status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_takes_part_in_autograd(layout, dtype, inverse):
    """Gradients through the operator are its other direction applied to the outputs' gradients, for q and k, alone or
    together, strided or expanded; where neither asks for one, nothing is recorded."""
    g = gen(12)
    table = al().rotary_table(60, 64, device=DEV, scaling={"type": "yarn", "factor": 2, "original": 30})
    pos = torch.randint(0, 60, (2, 7), generator=g).to(DEV)
    pos[0, 0] = -1
    q = torch.randn(2, 7, 5, 128, generator=g).to(TYPES[dtype]).to(DEV).transpose(1, 2).requires_grad_()
    k = torch.randn(2, 3, 7, 128, generator=g).to(TYPES[dtype]).to(DEV).requires_grad_()
    wq, wk = torch.randn(2, 5, 7, 128, generator=g).to(DEV), torch.randn(2, 3, 7, 128, generator=g).to(DEV)
    wq, wk = wq.to(TYPES[dtype]), wk.to(TYPES[dtype])
    kw = dict(layout=layout, inverse=inverse)
    back = dict(layout=layout, inverse=not inverse)
    plain = al().rotary_embed(q.detach(), k.detach(), table, pos, **kw)
    qo, ko = al().rotary_embed(q, k, table, pos, **kw)
    assert torch.equal(qo, plain[0]) and torch.equal(ko, plain[1])
    gq, gk = torch.autograd.grad([qo, ko], [q, k], [wq, wk])
    want = al().rotary_embed(wq, wk, table, pos, **back)
    assert torch.equal(gq, want[0]) and torch.equal(gk, want[1])
    assert torch.all(gq[0, :, 0] == 0)
    # one of the two; an expanded gradient (that of a sum); q alone
    only = torch.autograd.grad(al().rotary_embed(q.detach(), k, table, pos, **kw)[1].sum(), k)[0]
    assert torch.equal(only, al().rotary_embed(torch.ones_like(wk), None, table, pos, **back)[0])
    alone, none = al().rotary_embed(q, None, table, pos, **kw)
    assert none is None and torch.equal(torch.autograd.grad(alone, q, wq)[0], want[0])
    with torch.no_grad():
        assert not al().rotary_embed(q, k, table, pos, **kw)[0].requires_grad
    assert not plain[0].requires_grad and status() == 0


def test_rotary_gradient_against_differences_through_autograd():
    """Central differences of a loss through the operator; the map is linear, so a step of one has no truncation error."""
    g = gen(3)
    table = al().rotary_table(40, 96, device=DEV)
    x = torch.randn(1, 2, 2, 128, generator=g).to(DEV).requires_grad_()
    w = torch.randn(1, 2, 2, 128, generator=g).to(DEV)
    loss = lambda y: (al().rotary_embed(y, None, table, 9)[0].double() * w.double()).sum(dim=(1, 2, 3))
    loss(x).sum().backward()
    probe = torch.eye(512, device=DEV).view(512, 1, 2, 2, 128)
    with torch.no_grad():
        diff = torch.stack([(loss(x + p) - loss(x - p))[0] / 2 for p in probe])
    assert float((diff - x.grad.double().view(-1)).abs().max()) < 64 * 2 ** -23


def test_rotary_positions_are_checked():
    table = al().rotary_table(10, 128, device=DEV)
    q = torch.randn(2, 2, 3, 128, device=DEV)
    for at in (2 ** 63 - 1, 2 ** 63 - 3, 2 ** 62, 8, -1):
        with pytest.raises(ValueError, match="positions"):
            al().rotary_embed(q, None, table, at)
    for shape in ((4,), (2, 4), (3, 3), (2, 3, 1), (3, 1), (2, 1), (0,)):
        with pytest.raises(ValueError, match="positions"):
            al().rotary_embed(q, None, table, torch.zeros(shape, dtype=torch.int64, device=DEV))
    assert al().rotary_embed(q, None, table, 7)[0].shape == q.shape and status() == 0


def test_a_wrong_type_is_reported_by_name():
    c = al().Q8Cache.empty(1, 1, 64, DEV)
    x = torch.randn(1, 1, 3, 128, device=DEV)
    q = x[:, :, None]
    for call, name in ((lambda: al().append_q8(c, 3.5, x, x), "lengths"), (lambda: al().read_q8(c, "0", 3), "lo"),
                       (lambda: al().read_q8(c, 0, None), "hi"), (lambda: al().attend_q8(q, c, 3, window=1.5), "window"),
                       (lambda: al().attend_q8(q, c, 3, sinks=[]), "sinks"),
                       (lambda: al().attend_q8(q, c, torch.tensor([3], dtype=torch.int32, device=DEV), max_length="x"), "max_length"),
                       (lambda: al().attend_q8(q, c, 3, scale="x"), "scale"),
                       (lambda: al().rotary_embed(x, None, al().rotary_table(8, device=DEV), 0.5), "positions")):
        with pytest.raises(TypeError, match=name):
            call()
    for call, name in ((lambda: al().append_q8(c, 2 ** 70, x, x), "lengths"), (lambda: al().read_q8(c, -2 ** 70, 3), "lo"),
                       (lambda: al().attend_q8(q, c, 3, window=2 ** 31), "window"), (lambda: al().attend_q8(q, c, 3, sinks=2 ** 64), "sinks")):
        with pytest.raises(ValueError, match=name):
            call()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(4, 1), (2, 90)])
@pytest.mark.parametrize("gap", [0, 10, 16, 20, 28, 40, 100])
def test_quiet_blocks_under_a_loud_one(dtype, h, T, gap):
    """One block whose V is 2^gap louder than the others but zero in half of the dimensions: in those an output comes from
    the quiet blocks alone, and holds what the weights' lower end leaves of them (an absolute bound, relative to the row's
    loudest visible term), while the denominator counts every block in full."""
    n = 300
    cache = random_cache(gap, 1, 2, n)
    cache.v_exp.fill_(-50)
    cache.v_exp[..., 2] = gap - 50
    cache.v.view(torch.uint8)[:, :, 128:192, 64:] = 0
    q = make_q(gap + 1, 1, 2, h, T, dtype)
    out = host(al().attend_q8(q, cache, n)).astype(np.float64)
    one_term = dtype == "bf16" and T > 1
    for g in range(2):
        want, tol = q8_bounds.attend(host(q)[0, g].astype(np.float64), ref.values(host(cache.k), cache.k_exp.cpu().numpy())[0, g],
                                     host(cache.v)[0, g], cache.v_exp.cpu().numpy()[0, g], n, 0, 0, 1 / math.sqrt(128),
                                     terms=1 if one_term else 2, out_half_ulp=2 ** -8 if dtype == "bf16" else 2 ** -24)
        err = np.abs(out[0, g] - want)
        assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())
        if gap <= 10:                                                  # and there something of them is left
            assert np.abs(out[0, g][..., 64:] - want[..., 64:]).max() < 2 ** -6 * np.abs(want[..., 64:]).max()


@pytest.mark.parametrize("h, T", [(17, 1), (1, 40), (5, 4), (64, 2), (9, 3)])
def test_16_bit_queries_over_few_tokens_keep_two_terms(h, T):
    """Up to 128 rows over few tokens take the single tokens' kernel, whose weights are two f16 terms in either type: scores
    small enough that a lost low term shows (q8_bounds plants one on the CPU)."""
    n = 24
    cache = random_cache(h * T, 2, 1, 64)
    q = make_q(h, 2, 1, h, T, "bf16")
    out = host(al().attend_q8(q, cache, n, scale=0.02)).astype(np.float64)
    for b in range(2):
        want, tol = q8_bounds.attend(host(q)[b, 0].astype(np.float64), ref.values(host(cache.k), cache.k_exp.cpu().numpy())[b, 0],
                                     host(cache.v)[b, 0], cache.v_exp.cpu().numpy()[b, 0], n, 0, 0, 0.02, terms=2,
                                     out_half_ulp=2 ** -8)
        assert np.all(np.abs(out[b, 0] - want) <= tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_runs_of_zero_values(dtype):
    """Blocks whose V is all zero have the lowest exponent, so each of their tokens counts 2^100 times its weight in the
    denominator until a block with values comes: a CTA that walks 20000 of them alone, at weights just under the point
    where the maximum would follow, must not overflow there. Scores are 0 but for the first 64 tokens, 7.8 binades below."""
    B, G, h, T, n = 8, 19, 2, 80, 20000
    cache = al().Q8Cache.empty(B, G, n, DEV)
    cache.k.view(torch.uint8).zero_(), cache.v.view(torch.uint8).zero_()
    cache.k.view(torch.uint8)[:, :, :64, 0] = 0xB8                     # -1
    cache.k_exp.zero_(), cache.v_exp.fill_(-100)
    cache.v.view(torch.uint8)[:, :, 19968:] = 0x38                     # 1
    cache.v_exp[:, :, 19968 // 64:] = 0
    q = torch.zeros(B, G, h, T, 128, device=DEV, dtype=TYPES[dtype])
    q[..., 0] = 1.0
    scale = 7.8 * math.log(2)
    out = al().attend_q8(q, cache, n, scale=scale).double().cpu()
    p = torch.arange(n - T, n, dtype=torch.float64)                    # a query sees p + 1 tokens, p - 19967 with values
    want = (p - 19967).clamp(min=0) / (p + 1 - 64 + 64 * 2 ** -7.8)
    assert status() == 0
    # the weights are equal but for their rounding, which no sum here can hide: a part in 2^8 (16 bits) or 2^12
    tol = want * (2 ** -8 + 2 ** -12 if dtype == "bf16" else 2 ** -12)
    assert ((out - want[:, None]).abs() <= tol[:, None]).all()
