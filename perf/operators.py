"""Cases for measuring the 8-bit cache's operators: rotary positions, quantising a cache as it is written, reading it
back, and attention over it (single tokens and prompts, sliding window with sinks).

The cache of one layer holds K and V as e4m3 codes [B,G,C,128] and, for each block of 64 tokens of each (batch, group),
a power-of-two exponent [B,G,ceil(C/64)] (int8): value = code * 2^exponent. The shapes are the repository's own (32/8
and 16/8 heads of 128, contexts 2048 to 131072, prompts of 8192, a prefix of 4 tokens that stays visible) or odd ones.

`own = False` computes every operator in its plain form (elementary torch operations in 32 bits, rounded once at the
end); `own = True` calls the operators of attention_lab_b200.
"""
import math

import torch

own = False

D = 128            # head dimension
BLOCK = 64         # tokens that share one exponent
TOP = 448.0        # largest e4m3 value
E_MIN, E_MAX = -100, 120
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 32 requests, 32/8 heads: positions differ from request to request
        dict(name="rotary_token", op="rotary", B=32, T=1, Hq=32, Hk=8, rot=128, layout="half", inverse=False,
             dtype="bf16", table=32768, factor=1.0),
        # the gradient of a long batch's rotation, interleaved pairs, half of each head rotated, contexts stretched by 4
        dict(name="rotary_gradient_long", op="rotary", B=2, T=8191, Hq=32, Hk=8, rot=64, layout="interleaved",
             inverse=True, dtype="f32", table=131072, factor=4.0),
        # one decode step's write: 32 requests of different lengths, rotated on the way in
        dict(name="append_token", op="append", B=32, G=8, h=4, T=1, C=4096, low=1, high=4096, rope=True, rot=128,
             layout="half", dtype="bf16"),
        # a prompt chunk of 8192 tokens written behind 2048 earlier ones that end inside a block
        dict(name="append_prompt", op="append", B=1, G=8, h=4, T=8192, C=16384, low=10270, high=10270, rope=True,
             rot=128, layout="half", dtype="bf16"),
        # a few rows of a short cache, read back in 32 bits between odd positions
        dict(name="read_rows", op="read", B=3, G=2, C=515, lo=61, hi=450, dtype="f32"),
        # a whole 128K context read back for the 16-bit operators
        dict(name="read_context", op="read", B=1, G=8, C=131072, lo=0, hi=131072, dtype="bf16"),
        # the smallest decode step: one request, 16/8 heads, 2048 tokens
        dict(name="token_short", op="attend", B=1, G=8, h=2, T=1, C=2048, low=2048, high=2048, window=0, sinks=0,
             dtype="bf16"),
        # the batch decode step: 32 requests between 16K and 32K tokens, 32/8 heads
        dict(name="token_batch", op="attend", B=32, G=8, h=4, T=1, C=32768, low=16384, high=32768, window=0, sinks=0,
             dtype="bf16"),
        # long contexts of which 4 first tokens and the last 4096 stay visible, 32 bits
        dict(name="token_window", op="attend", B=6, G=8, h=4, T=1, C=65536, low=100, high=65536, window=4096, sinks=4,
             dtype="f32"),
        # a ragged batch of short prompts, padded on the left, 32 bits, three heads to a group
        dict(name="prompt_ragged", op="attend", B=5, G=2, h=3, T=333, C=700, low=201, high=641, window=0, sinks=0,
             dtype="f32"),
        # a chunk of 1024 tokens late in two 16K contexts, sliding window and sinks
        dict(name="prompt_window", op="attend", B=2, G=8, h=4, T=1024, C=16384, low=15001, high=16384, window=2048,
             sinks=4, dtype="bf16"),
        # a whole prompt of 8192 tokens
        dict(name="prompt_full", op="attend", B=1, G=8, h=4, T=8192, C=8192, low=8192, high=8192, window=0, sinks=0,
             dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(max(n, lo), hi)
    return n - 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["rotary", "append", "read", "token", "prompt"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    layout = rng.choice(["half", "interleaved"])
    rot = rng.choice([128, 128, 64, 96, 32, 20])
    if op == "rotary":
        B = _spread(rng, 1, 32)
        T = _spread(rng, 1, max(1, 16384 // B))
        return dict(op=op, B=B, T=T, Hq=rng.choice([1, 6, 8, 16, 32]), Hk=rng.choice([1, 2, 8]), rot=rot,
                    layout=layout, inverse=rng.random() < 0.5, dtype=dtype, table=T + _spread(rng, 1, 100000),
                    factor=rng.choice([1.0, 2.0, 4.0]))
    if op == "append":
        B = _spread(rng, 1, 32)
        G = rng.choice([1, 2, 8])
        T = 1 if rng.random() < 0.4 else _spread(rng, 2, max(2, 8192 // B))
        low = _spread(rng, 1, T + 1000)
        high = low + _spread(rng, 1, 1000)
        return dict(op=op, B=B, G=G, h=rng.choice([1, 2, 3, 4]), T=T, C=max(high, T) + rng.randrange(0, 200), low=low,
                    high=high, rope=rng.random() < 0.7, rot=rot, layout=layout, dtype=dtype)
    if op == "read":
        B, G = _spread(rng, 1, 16), rng.choice([1, 2, 8])
        C = _spread(rng, 64, max(64, (1 << 20) // (B * G)))
        lo = rng.randrange(0, C)
        return dict(op=op, B=B, G=G, C=C, lo=lo, hi=rng.randrange(lo + 1, C + 1), dtype=dtype)
    window, sinks = (_spread(rng, 16, 8192), rng.choice([0, 1, 4, 64, 100])) if rng.random() < 0.5 else (0, 0)
    G = rng.choice([1, 2, 8])
    if op == "token":
        B, h = _spread(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8])
        C = _spread(rng, 16, min(131072, (1 << 23) // (B * G)))
        high = rng.randrange(max(1, C // 2), C + 1)
        return dict(op="attend", B=B, G=G, h=h, T=rng.choice([1, 1, 1, 2]), C=C, low=rng.randrange(1, high + 1), high=high,
                    window=window, sinks=sinks, dtype=dtype)
    B, h = _spread(rng, 1, 4), rng.choice([1, 2, 3, 4, 8])
    T = _spread(rng, 9, 8192)
    most = min(32768, 1_000_000_000 // (B * G * h * T))
    C = max(T, _spread(rng, 64, max(64, most)))
    while B * G * h * T * C > 2_000_000_000:
        T = T // 2
        C = max(T, C // 2)
    high = rng.randrange(max(1, C // 2), C + 1)
    return dict(op="attend", B=B, G=G, h=h, T=T, C=C, low=rng.randrange(max(1, high // 2), high + 1), high=high,
                window=window, sinks=sinks, dtype=dtype)


def _lengths(case):
    """The requests' lengths, between the case's low and high, in an order that is not sorted."""
    B, low, high = case["B"], case["low"], case["high"]
    if B == 1:
        return [high]
    step = next(s for s in (7, 11, 13, 17) if math.gcd(s, B) == 1)
    return [low + (high - low) * (i * step % B) // (B - 1) for i in range(B)]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _features(gen, B, G, n, keys):
    """Rows as a layer makes them: tokens of different size and, for keys, a few channels far above the others."""
    x = _normal(gen, B, G, n, D)
    x *= torch.exp(0.5 * _normal(gen, B, G, n, 1))
    if keys:
        x *= torch.where(torch.rand(1, G, 1, D, generator=gen, device=DEV) < 0.04, 6.0, 1.0)
    return x


def _table(length, rot, factor):
    """Rotary table [length, rot]: cosines, then sines, of position * frequency; the frequencies below one turn in the
    original context are divided by `factor`, those above a few dozen turns kept, with a ramp between."""
    i = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    freq = 1e6 ** (-2.0 * i / rot)
    if factor != 1.0:
        turns = freq * (length / factor) / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        freq = freq * keep + freq / factor * (1.0 - keep)
    amp = 1.0 if factor == 1.0 else 0.1 * math.log(factor) + 1.0
    ang = torch.arange(length, device=DEV, dtype=torch.float64)[:, None] * freq
    return torch.cat([ang.cos() * amp, ang.sin() * amp], dim=1).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    op, dt = case["op"], _TYPES[case["dtype"]] if "dtype" in case else None
    s = dict(case=case)
    B = case["B"]
    if op == "rotary":
        T = case["T"]
        s["q"] = _normal(gen, B, T, case["Hq"], D).to(dt).transpose(1, 2)
        s["k"] = _normal(gen, B, T, case["Hk"], D).to(dt).transpose(1, 2)
        first = torch.randint(0, case["table"] - T + 1, (B, 1), generator=gen, device=DEV)
        s["positions"] = first + torch.arange(T, device=DEV)
        s["table"] = _table(case["table"], case["rot"], case["factor"])
        return s
    G, C = case["G"], case["C"]
    for name, keys in (("k", True), ("v", False)):
        codes, exps = _quantise_blocks(_features(gen, B, G, C, keys))
        s[name], s[name + "_exp"] = codes, exps
    if op == "read":
        return s
    T, h = case["T"], case["h"]
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV)
    if op == "append":
        s["k_new"] = _features(gen, B, G, T, True).to(dt)
        s["v_new"] = _features(gen, B, G, T, False).to(dt)
        if case["rope"]:
            s["q"] = _normal(gen, B, T, G, h, D).to(dt).permute(0, 2, 3, 1, 4)
            s["table"] = _table(C, case["rot"], 1.0)
    else:
        s["q"] = _normal(gen, B, T, G, h, D).to(dt).permute(0, 2, 3, 1, 4)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, from the bits of amax (32 bits)."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > TOP / 512.0).to(x.dtype)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX)


def _power(e):
    """2^e in 32 bits, from its bits (a library power may be an ulp off)."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _codes(x, e):
    """Codes of x under the exponents e, to the nearest, ties to even."""
    return (x * _power(-e)).to(torch.float8_e4m3fn)


def _quantise_blocks(x):
    """Whole blocks of a new cache [B,G,C,d] -> codes, exponents."""
    B, G, C, d = x.shape
    nb = -(-C // BLOCK)
    x = torch.cat([x, x.new_zeros(B, G, nb * BLOCK - C, d)], dim=2).view(B, G, nb, BLOCK, d)
    e = _exponent(x.abs().amax(dim=(3, 4)))
    codes = _codes(x, e[..., None, None]).view(B, G, nb * BLOCK, d)[:, :, :C].contiguous()
    return codes, e.to(torch.int8)


def _values(codes, exps):
    """codes * 2^exponent of the token's block, in 32 bits."""
    scale = _power(exps).repeat_interleave(BLOCK, dim=2)[:, :, :codes.shape[2], None]
    return codes.float() * scale


def _rotate(x, cos, sin, layout, inverse):
    """x [..., d] in 32 bits, cos / sin [..., rot/2] broadcast to it; dimensions past rot are passed through."""
    half = cos.shape[-1]
    if inverse:
        sin = -sin
    if layout == "half":
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_rotary(s):
    c = s["case"]
    half = c["rot"] // 2
    rows = s["table"][s["positions"]][:, None]                                   # [B,1,T,rot]
    return tuple(_rotate(x.float(), rows[..., :half], rows[..., half:], c["layout"], c["inverse"]).to(x.dtype)
                 for x in (s["q"], s["k"]))


def _write(codes, exps, new, lengths):
    """The append of one tensor: row t of `new` (32 bits) goes to position lengths - T + t (dropped below 0). A block
    that keeps earlier rows keeps at least its exponent; where that grows, the kept rows are rounded again."""
    B, G, C, d = codes.shape
    T = new.shape[2]
    start = lengths.long() - T                                                   # [B]
    first = start.clamp(min=0) // BLOCK
    nb = -(-C // BLOCK)
    touched = min((T - 1) // BLOCK + 2, nb)
    block = first[:, None] + torch.arange(touched, device=DEV)                   # [B,n]
    ok = block * BLOCK < lengths[:, None]
    pos = block[:, :, None] * BLOCK + torch.arange(BLOCK, device=DEV)            # [B,n,64]
    t = pos - start[:, None, None]
    fresh = (t >= 0) & (t < T) & (pos < C) & ok[:, :, None]
    kept = (t < 0) & ok[:, :, None]
    bi = torch.arange(B, device=DEV)
    x = new[bi[:, None, None], :, t.clamp(0, T - 1)].permute(0, 3, 1, 2, 4)      # [B,G,n,64,d]
    x = torch.where(fresh[:, None, :, :, None], x, 0.0)
    at = pos.clamp(max=C - 1)
    old = codes.view(torch.uint8)[bi[:, None, None], :, at].permute(0, 3, 1, 2, 4)
    eb = block.clamp(max=nb - 1)
    e_old = exps[bi[:, None], :, eb].permute(0, 2, 1).int()                      # [B,G,n]
    e_new = _exponent(x.abs().amax(dim=(3, 4)))
    has_kept = kept.any(dim=2)[:, None]
    e = torch.where(has_kept, torch.maximum(e_old, e_new), e_new)
    again = _codes(old.contiguous().view(torch.float8_e4m3fn).float(), (e - e_old)[..., None, None])
    again = torch.where(kept[:, None, :, :, None], again.view(torch.uint8), old)
    put = torch.where(fresh[:, None, :, :, None], _codes(x, e[..., None, None]).view(torch.uint8), again)
    b_, n_, r_ = torch.nonzero(fresh | (kept & (pos < C)), as_tuple=True)
    codes.view(torch.uint8)[b_, :, pos[b_, n_, r_]] = put[b_, :, n_, r_]
    b_, n_ = torch.nonzero(fresh.any(dim=2), as_tuple=True)
    exps[b_, :, block[b_, n_]] = e[b_, :, n_].to(torch.int8)


def _plain_append(s):
    c = s["case"]
    k, v, q = s["k_new"].float(), s["v_new"].float(), None
    if c["rope"]:
        half, T = c["rot"] // 2, c["T"]
        pos = s["lengths"].long()[:, None] - T + torch.arange(T, device=DEV)     # [B,T]
        rows = s["table"][pos.clamp(min=0)]
        cos, sin = rows[..., :half], rows[..., half:]
        k = _rotate(k, cos[:, None], sin[:, None], c["layout"], False)
        q = _rotate(s["q"].float(), cos[:, None, None], sin[:, None, None], c["layout"], False)
        q = torch.where(pos[:, None, None, :, None] >= 0, q, 0.0).to(s["q"].dtype)
    _write(s["k"], s["k_exp"], k, s["lengths"])
    _write(s["v"], s["v_exp"], v, s["lengths"])
    return q


def _plain_attend(s):
    c = s["case"]
    B, G, h, T, d = s["q"].shape
    C = c["C"]
    k = _values(s["k"], s["k_exp"])
    scores = torch.matmul(s["q"].float().reshape(B, G, h * T, d), k.transpose(2, 3)) / math.sqrt(d)
    del k
    pos = (s["lengths"].long()[:, None] - T + torch.arange(T, device=DEV))[:, :, None]   # [B,T,1]
    j = torch.arange(C, device=DEV)
    seen = (j <= pos) if c["window"] == 0 else (j <= pos) & ((j > pos - c["window"]) | (j < c["sinks"]))
    scores = scores.view(B, G, h, T, C).masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(scores.sub_(top))
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.view(B, G, h * T, C), _values(s["v"], s["v_exp"])).view(B, G, h, T, d)
    return torch.where(total > 0, out / total, 0.0).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        import attention_lab_b200 as al
        if op == "rotary":
            return al.rotary_embed(s["q"], s["k"], s["table"], s["positions"], layout=c["layout"], inverse=c["inverse"])
        cache = al.Q8Cache(s["k"], s["v"], s["k_exp"], s["v_exp"])
        if op == "append":
            q = al.append_q8(cache, s["lengths"], s["k_new"], s["v_new"], q=s.get("q"), table=s.get("table"),
                             layout=c["layout"])
        elif op == "read":
            return al.read_q8(cache, c["lo"], c["hi"], dtype=_TYPES[c["dtype"]])
        else:
            return al.attend_q8(s["q"], cache, s["lengths"], window=c["window"], sinks=c["sinks"])
    elif op == "rotary":
        return _plain_rotary(s)
    elif op == "append":
        q = _plain_append(s)
    elif op == "read":
        return tuple(_values(s[n][:, :, :c["hi"]], s[n + "_exp"])[:, :, c["lo"]:].to(_TYPES[c["dtype"]])
                     for n in ("k", "v"))
    else:
        return _plain_attend(s)
    got = dict(k=s["k"], v=s["v"], k_exp=s["k_exp"], v_exp=s["v_exp"])
    return got if q is None else dict(got, q=q)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    op, B = case["op"], case["B"]
    es = 2 if case["dtype"] == "bf16" else 4
    if op == "rotary":
        heads, tokens = case["Hq"] + case["Hk"], B * case["T"]
        return dict(bytes=tokens * (heads * D * es * 2 + case["rot"] * 4 + 8), flops=tokens * heads * case["rot"] * 3)
    G = case["G"]
    if op == "read":
        rows = B * G * (case["hi"] - case["lo"])
        return dict(bytes=2 * rows * (D * (1 + es) + 1 / BLOCK), flops=2 * rows * D)
    T, h = case["T"], case["h"]
    if op == "append":
        rows = sum(min(T, n) for n in _lengths(case))
        moved = rows * G * 2 * (D * (es + 1) + 1 / BLOCK)
        flops = rows * G * 2 * D * 2
        if case["rope"]:
            moved += rows * (G * h * D * es * 2 + case["rot"] * 4)
            flops += rows * G * (h + 1) * case["rot"] * 3
        return dict(bytes=moved, flops=flops)
    window, sinks = case["window"], case["sinks"]
    rows = pairs = 0
    for n in _lengths(case):
        first = max(n - T, 0)
        left = max(first - window + 1, 0) if window else 0
        rows += n - left + min(sinks if window else 0, left)
        for p in range(first, n):
            left = max(p - window + 1, 0) if window else 0
            pairs += p + 1 - left + min(sinks if window else 0, left)
    return dict(bytes=rows * G * 2 * (D + 1 / BLOCK) + 2 * B * G * h * T * D * es, flops=pairs * G * h * D * 4)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_turn(x, angle_cos, angle_sin, layout):
    """Each pair as a complex number times (cos + i sin)."""
    half = angle_cos.shape[-1]
    z = torch.complex(x[..., :half], x[..., half:2 * half]) if layout == "half" else \
        torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    z = z * torch.complex(angle_cos, angle_sin)
    y = x.clone()
    if layout == "half":
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
    else:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
    return y


def _exact_power(e):
    """2^e in 64 bits for whole e, looked up: a library power may be an ulp off."""
    powers = torch.tensor([2.0 ** i for i in range(-256, 257)], dtype=torch.float64, device=DEV)
    return powers[e.long() + 256]


def _exact_grid(x):
    """The nearest e4m3 value: 3 bits after the leading one, steps of 2^-9 below 2^-6, ties to even."""
    step = _exact_power(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)
    return torch.round(x / step) * step


def _exact_append(codes, exps, new, lengths):
    codes, T = codes.double(), new.shape[2]
    for b, n in enumerate(lengths):
        start = max(n - T, 0)
        for at in range(start // BLOCK, -(-n // BLOCK)):
            lo, hi = max(at * BLOCK, start), min((at + 1) * BLOCK, n)
            x = new[b, :, lo - (n - T):hi - (n - T)]
            # the least e with amax <= 448 * 2^e; log2 of an exact power of two may come out an ulp high
            e = torch.ceil(torch.log2(x.abs().amax(dim=(1, 2)) / TOP) - 1e-12).clamp(E_MIN, E_MAX)
            if at * BLOCK < lo:
                before = exps[b, :, at].double()
                e = torch.maximum(e, before)
                old = codes[b, :, at * BLOCK:lo] * _exact_power(before - e)[:, None, None]
                codes[b, :, at * BLOCK:lo] = _exact_grid(old)
            codes[b, :, lo:hi] = _exact_grid(x * _exact_power(-e)[:, None, None])
    return codes


def _exact_attend(case, s):
    B, G, h, T, d = s["q"].shape
    out = torch.zeros(B, G, h, T, d, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_lengths(case)):
        skip = max(T - n, 0)
        at = torch.arange(n - T + skip, n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None, :]
        hidden = j > at
        if case["window"]:
            hidden = hidden | ((at - j >= case["window"]) & (j >= case["sinks"]))
        for g in range(G):
            kv = []
            for name in ("k", "v"):
                e = s[name + "_exp"][b, g, torch.arange(n, device=DEV) // BLOCK].double()
                kv.append(s[name][b, g, :n].double() * _exact_power(e)[:, None])
            for i in range(h):
                w = s["q"][b, g, i, skip:].double() @ kv[0].T / d ** 0.5
                w[hidden] = float("-inf")
                out[b, g, i, skip:] = torch.softmax(w, dim=1) @ kv[1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        rows = s["table"].double()[s["positions"]][:, None]
        half = case["rot"] // 2
        sin = rows[..., half:] * (-1.0 if case["inverse"] else 1.0)
        return tuple(_exact_turn(s[n].double(), rows[..., :half], sin, case["layout"]) for n in ("q", "k"))
    if op == "read":
        at = torch.arange(case["lo"], case["hi"], device=DEV)
        return tuple(s[n][:, :, case["lo"]:case["hi"]].double()
                     * _exact_power(s[n + "_exp"][:, :, at // BLOCK])[..., None] for n in ("k", "v"))
    if op == "attend":
        return _exact_attend(case, s)
    lengths, T = _lengths(case), case["T"]
    k, got = s["k_new"].double(), {}
    if case["rope"]:
        q, half = s["q"].double(), case["rot"] // 2
        for b, n in enumerate(lengths):
            skip = max(T - n, 0)
            rows = s["table"].double()[n - T + skip:n]
            k[b, :, skip:] = _exact_turn(k[b, :, skip:], rows[:, :half], rows[:, half:], case["layout"])
            q[b, :, :, skip:] = _exact_turn(q[b, :, :, skip:], rows[:, :half], rows[:, half:], case["layout"])
            q[b, :, :, :skip] = 0.0
        got["q"] = q
    got["k"] = _exact_append(s["k"], s["k_exp"], k, lengths)
    got["v"] = _exact_append(s["v"], s["v_exp"], s["v_new"].double(), lengths)
    return dict(got, k_exp=None, v_exp=None)
