"""Layer norm, rotary positions and attention on token sequences (diffphycon_amd.sequence) against their definitions in 64 bits, within the
error bounds that tests/sequence_oracle.py derives for each formula."""
import math
import random

import pytest
import torch

import sequence_oracle as O

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a real MI355X"
    return torch.device("cuda:0")


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0, dev="cuda:0"):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).to(dev)


def _within(name, got, value, bound):
    got, value, bound = got.double(), value.to(got.device), bound.to(got.device)
    same = (got == value) | (got.isnan() & value.isnan())
    off = torch.where(same, torch.zeros_like(bound), (got - value).abs() / bound.clamp_min(1e-300))
    worst = off.max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst} times its bound at {tuple(int(i) for i in torch.nonzero(off == off.max())[0]) if off.dim() else ()}"      # (NaN fails too)
    return worst


# ---------------------------------------------------------------------------------------------------------------- attention
def _check_attention(q, k, v, dout, out, lse, grads, lengths, packed=False, causal=False, scale=None, mask=None):
    """Every head of every sequence against the oracle; rows outside the sequences must be zero (lse: -inf)."""
    H, Hk = q.shape[-2], k.shape[-2]
    G, t = H // Hk, q.dtype
    seen_q, seen_k = torch.zeros(q.shape[:-2], dtype=torch.bool), torch.zeros(k.shape[:-2], dtype=torch.bool)
    q0 = k0 = 0
    for b, (nq, nk) in enumerate(lengths):
        qi, ki = (slice(q0, q0 + nq), slice(k0, k0 + nk)) if packed else ((b, slice(0, nq)), (b, slice(0, nk)))
        q0, k0 = q0 + nq, k0 + nk
        seen_q[qi], seen_k[ki] = True, True
        for hk in range(Hk):
            sums = None
            for h in range(hk * G, hk * G + G):
                r = O.attention(q[qi][:, h], k[ki][:, hk], v[ki][:, hk], dout[qi][:, h] if dout is not None else None, causal, scale, mask[ki] if mask is not None else None)
                _within("out", out[qi][:, h], *r["out"])
                _within("lse", lse[h, qi] if packed else lse[b, h, :nq], *r["lse"])
                if dout is not None:
                    _within("dq", grads[0][qi][:, h], r["dq"][0], O.add_rounding(*r["dq"], t))
                    part = [*r["dk"], *r["dv"]]
                    sums = part if sums is None else [x + y for x, y in zip(sums, part)]
            if dout is not None:                                     # (the sum over the group: one fp32 chain over all its rows)
                chain = G * O.E * nq
                _within("dk", grads[1][ki][:, hk], sums[0], O.add_rounding(sums[0], sums[1] * (1 + chain), t))
                _within("dv", grads[2][ki][:, hk], sums[2], O.add_rounding(sums[2], sums[3] * (1 + chain), t))
    if not packed:
        assert not out[~seen_q].any() and torch.isneginf(lse.transpose(1, 2)[~seen_q]).all()
        if dout is not None:
            assert not grads[0][~seen_q].any() and not grads[1][~seen_k].any() and not grads[2][~seen_k].any()


SHAPES = [
    # B, Lq, Lk, H, Hk, D, causal
    (1, 1, 1, 1, 1, 8, False), (3, 1, 1, 2, 1, 128, True), (2, 33, 33, 4, 2, 32, False), (2, 64, 64, 2, 2, 64, True), (1, 128, 128, 2, 1, 128, False),
    (1, 129, 65, 4, 4, 40, False), (2, 131, 70, 4, 2, 24, True),            # more queries than keys: the first rows see nothing
    (1, 5, 300, 6, 2, 64, True), (1, 1, 777, 8, 2, 128, False), (2, 7, 1000, 3, 3, 96, False), (1, 200, 511, 2, 2, 128, True), (1, 257, 191, 3, 3, 96, False),
    (1, 384, 640, 2, 1, 80, True), (6, 17, 17, 5, 5, 16, True), (1, 300, 1, 2, 2, 32, False), (1, 300, 1, 2, 2, 32, True), (40, 32, 32, 8, 8, 32, False),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_and_its_gradients(shape, t, dev):
    from diffphycon_amd import sequence as S
    B, Lq, Lk, H, Hk, D, causal = shape
    g = _gen(hash(shape) % 1000)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    out, lse = S.attention_forward(q, k, v, causal=causal)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal)
    _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)] * B, causal=causal)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("causal,Lq,Lk", [(False, 236, 1), (False, 236, 11), (False, 150, 47), (True, 90, 90)])
def test_attention_when_the_card_is_full(causal, Lq, Lk, D, t, dev):
    """Every place on the card is taken, by one sequence over and over: each copy gives the first one's results, to the bit."""
    from diffphycon_amd import sequence as S
    B, H, Hk = 160, 10, 5
    g = _gen(Lk + D)
    one = lambda L, h: _randn(g, 1, L, h, D, dtype=t).expand(B, L, h, D)  # noqa: E731
    q, k, v, dout = one(Lq, H), one(Lk, Hk), one(Lk, Hk), one(Lq, H)
    for _ in range(2):
        out, lse = S.attention_forward(q, k, v, causal=causal)
        grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal)
        for x in (out, lse, *grads):
            assert torch.equal(x, x[:1].expand_as(x))
    _check_attention(q[:1], k[:1], v[:1], dout[:1], out[:1], lse[:1], [x[:1] for x in grads], [(Lq, Lk)], causal=causal)


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
def test_attention_gradients_of_rows_with_few_keys(t, dev):
    """Short sequences beside long ones that are split: what the rounding of `out` loses in D must not reach dq, nor dk.  A row of one key has no
    gradient but dv's: what is left is fp32's rounding."""
    from diffphycon_amd import sequence as S
    ql, kl, H, D = [11, 4, 9, 1, 7], [961, 2, 61, 1, 250], 4, 64
    g = _gen(23)
    q, k, v, dout = _randn(g, sum(ql), H, D, dtype=t), _randn(g, sum(kl), H, D, dtype=t), _randn(g, sum(kl), H, D, dtype=t), _randn(g, sum(ql), H, D, dtype=t)
    plan = S.SequencePlan.packed(ql, kl, device=dev)
    out, lse = S.attention_forward(q, k, v, plan=plan)
    dq, dk, _ = S.attention_backward(dout, q, k, v, out, lse, plan=plan)
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        for h in range(H):
            a, b = (slice(q0, q0 + nq), h), (slice(k0, k0 + nk), h)
            r = O.attention(q[a], k[b], v[b], dout[a], swept=nk <= 256)
            _within("dq", dq[a], r["dq"][0], O.add_rounding(*r["dq"], t))
            _within("dk", dk[b], r["dk"][0], O.add_rounding(*r["dk"], t))
        q0, k0 = q0 + nq, k0 + nk


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
@pytest.mark.parametrize("D,causal", [(32, False), (64, True), (96, False), (128, True)])
def test_attention_gradients_of_short_sequences_round_once(D, causal, t, dev):
    """Sums of few terms do not average their operands' roundings: they take P and dS in two parts."""
    from diffphycon_amd import sequence as S
    ql, kl, H, Hk = [2, 7, 32, 1, 20, 3] + ([400] if causal else []), [2, 5, 64, 40, 33, 4] + ([3] if causal else []), 4, 2
    g = _gen(41 + D)
    q, k, v, dout = _randn(g, sum(ql), H, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(ql), H, D, dtype=t)
    plan = S.SequencePlan.packed(ql, kl, device=dev)
    out, lse = S.attention_forward(q, k, v, causal=causal, plan=plan)
    dq, dk, dv = S.attention_backward(dout, q, k, v, out, lse, causal=causal, plan=plan)
    q0 = k0 = 0
    for nq, nk in zip(ql, kl):
        for hk in range(Hk):
            b, sums = (slice(k0, k0 + nk), hk), None
            for h in range(hk * 2, hk * 2 + 2):
                a = (slice(q0, q0 + nq), h)
                r = O.attention(q[a], k[b], v[b], dout[a], causal, swept=True, parts=True)
                _within("dq", dq[a], r["dq"][0], O.add_rounding(*r["dq"], t))
                part = [*r["dk"], *r["dv"]]
                sums = part if sums is None else [x + y for x, y in zip(sums, part)]
            chain = 2 * O.E * nq
            _within("dk", dk[b], sums[0], O.add_rounding(sums[0], sums[1] * (1 + chain), t))
            _within("dv", dv[b], sums[2], O.add_rounding(sums[2], sums[3] * (1 + chain), t))
        q0, k0 = q0 + nq, k0 + nk


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_of_one_key_has_no_gradient_but_the_values(t, dev):
    """The softmax of one key is 1 whatever the query and the key: their gradients are zero, not the rounding of P (dP - D)."""
    from diffphycon_amd import sequence as S
    g = _gen(31)
    q, dout = _randn(g, 3, 40, 6, 80, dtype=t), _randn(g, 3, 40, 6, 80, dtype=t)
    k, v = _randn(g, 3, 1, 2, 80, dtype=t), _randn(g, 3, 1, 2, 80, dtype=t)
    out, lse = S.attention_forward(q, k, v)
    dq, dk, dv = S.attention_backward(dout, q, k, v, out, lse)
    assert not dq.any() and not dk.any()
    _check_attention(q, k, v, dout, out, lse, (dq, dk, dv), [(40, 1)] * 3)
    plan = S.SequencePlan.packed([40, 40, 40], [1, 0, 2], device=dev)
    q, k, v, dout = q.reshape(120, 6, 80), k.reshape(3, 2, 80), v.reshape(3, 2, 80), dout.reshape(120, 6, 80)
    out, lse = S.attention_forward(q, k, v, plan=plan)
    grads = S.attention_backward(dout, q, k, v, out, lse, plan=plan)
    assert not grads[0][:80].any() and grads[0][80:].any() and not grads[1][0].any() and grads[1][1:].any()
    _check_attention(q, k, v, dout, out, lse, grads, [(40, 1), (40, 0), (40, 2)], packed=True)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_masks(t, causal, dev):
    """Padded keys hold infinities and NaN; one batch entry has no key at all; one has holes."""
    from diffphycon_amd import sequence as S
    B, Lq, Lk, H, Hk, D = 4, 70, 150, 4, 2, 48
    g = _gen(5)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    mask = torch.ones(B, Lk, dtype=torch.bool)
    mask[1, 40:] = False
    mask[2] = False
    mask[3] = torch.rand(Lk, generator=g) < 0.5
    mask[3, :90] = False                                             # with the causal mask the first rows see nothing
    mask = mask.to(dev)
    for x, bad in ((k, math.nan), (v, math.inf)):
        x[~mask] = bad
    k[~mask & (torch.arange(Lk, device=dev)[None] % 2 == 0)] = -math.inf
    dead = torch.zeros(B, Lq, dtype=torch.bool, device=dev)
    dead[2] = True
    if causal:
        dead[3, :10] = True
    q[dead], dout[dead] = math.nan, math.inf                          # rows that see nothing take no part, whatever they hold
    out, lse = S.attention_forward(q, k, v, causal=causal, key_mask=mask)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, key_mask=mask)
    assert torch.isneginf(lse[2]).all() and not out[dead].any()
    q, dout = q.masked_fill(dead[:, :, None, None], 0.0), dout.masked_fill(dead[:, :, None, None], 0.0)
    _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)] * B, causal=causal, mask=mask)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("Lq,D,causal", [(150, 64, True), (70, 128, False), (5, 64, True), (300, 32, False)])
def test_attention_masks_with_holes_of_whole_tiles(Lq, D, causal, t, dev):
    """Tiles and blocks that no key takes part in are left out: between others, first, last, and all of them."""
    from diffphycon_amd import sequence as S
    B, Lk, H, Hk = 5, 900, 4, 2
    g = _gen(61 + Lq)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    mask = torch.ones(B, Lk, dtype=torch.bool)
    mask[0, :400] = False
    mask[1, 64:700] = False
    mask[2, 130:] = False
    mask[3] = torch.rand(Lk // 50, generator=g).repeat_interleave(50) < 0.3
    mask[4] = False
    mask[4, 640] = True
    mask = mask.to(dev)
    k[~mask], v[~mask] = math.nan, -math.inf
    out, lse = S.attention_forward(q, k, v, causal=causal, key_mask=mask)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, key_mask=mask)
    _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)] * B, causal=causal, mask=mask)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_packed(t, causal, dev):
    from diffphycon_amd import sequence as S
    ql, kl = [130, 0, 1, 64, 33, 5, 200], [130, 7, 1, 0, 257, 3, 90]
    H, Hk, D = 4, 2, 64
    g = _gen(7)
    q, k, v, dout = _randn(g, sum(ql), H, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(ql), H, D, dtype=t)
    mask = (torch.rand(sum(kl), generator=g) < 0.8).to(dev)
    plan = S.SequencePlan.packed(ql, kl, device=dev)
    for m in (None, mask):
        out, lse = S.attention_forward(q, k, v, causal=causal, plan=plan, key_mask=m)
        grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, plan=plan, key_mask=m)
        _check_attention(q, k, v, dout, out, lse, grads, list(zip(ql, kl)), packed=True, causal=causal, mask=m)


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_padded(t, dev):
    """Rows behind a sequence hold NaN and do not matter; outputs there are zero, or untouched in the caller's buffers."""
    from diffphycon_amd import sequence as S
    ql, kl, H, D = [50, 0, 129, 7], [50, 20, 100, 0], 2, 32
    B, Lq, Lk = 4, 140, 120
    g = _gen(8)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    for b in range(B):
        q[b, ql[b]:], dout[b, ql[b]:], k[b, kl[b]:], v[b, kl[b]:] = math.nan, math.nan, math.nan, math.inf
    plan = S.SequencePlan.padded(ql, Lq, kl, Lk, device=dev)
    out, lse = S.attention_forward(q, k, v, causal=True, plan=plan)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=True, plan=plan)
    _check_attention(q, k, v, dout, out, lse, grads, list(zip(ql, kl)), causal=True)
    buf = torch.full_like(out, 7.0)
    S.attention_forward(q, k, v, causal=True, plan=plan, out=buf)
    bufs = [torch.full_like(x, 7.0) for x in grads]
    S.attention_backward(dout, q, k, v, out, lse, causal=True, plan=plan, grads=bufs)
    for b in range(B):
        assert (buf[b, ql[b]:] == 7).all() and torch.equal(buf[b, :ql[b]], out[b, :ql[b]])
        for x, y, n in zip(bufs, grads, (ql[b], kl[b], kl[b])):
            assert (x[b, n:] == 7).all() and torch.equal(x[b, :n], y[b, :n])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_attention_layouts(t, dev):
    """Views of one projection, heads before tokens, an odd base, broadcast keys: all equal to contiguous inputs, bit for bit."""
    from diffphycon_amd import sequence as S
    B, L, H, D = 2, 77, 3, 32
    g = _gen(9)
    qkv, dout = _randn(g, B, L, 3, H, D, dtype=t), _randn(g, B, H, L, D, dtype=t).transpose(1, 2)
    q, k, v = qkv.unbind(2)
    c = [x.contiguous() for x in (q, k, v, dout)]
    out, lse = S.attention_forward(*c[:3], causal=True)
    ref = S.attention_backward(c[3], *c[:3], out, lse, causal=True)
    out2, lse2 = S.attention_forward(q, k, v, causal=True)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    d = torch.empty_like(qkv)
    got = S.attention_backward(dout, q, k, v, out2, lse2, causal=True, grads=d.unbind(2))
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    odd = torch.empty(q.numel() + 1, dtype=t, device=dev)[1:].view(q.shape)
    odd.copy_(q)
    out3, _ = S.attention_forward(odd, k, v, causal=True)
    assert torch.equal(out, out3)
    one = _randn(g, 1, L, 1, D, dtype=t)
    wide = one.expand(B, L, H, D)
    o1, l1 = S.attention_forward(q, wide, wide)
    o2, l2 = S.attention_forward(q, wide.contiguous(), wide.contiguous())
    assert torch.equal(o1, o2)
    for a, b in zip(S.attention_backward(dout, q, wide, wide, o1, l1), S.attention_backward(dout, q, wide.contiguous(), wide.contiguous(), o2, l2)):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        S.attention_forward(q, k, v, out=q)
    with pytest.raises(ValueError):
        S.attention_backward(dout, q, k, v, out, lse, causal=True, grads=(d[:, :, 0], d[:, :, 1], d[:, :, 1]))


def test_attention_gradient_against_differences(dev):
    """Directional derivatives of sum(out w) by central differences of the 64-bit definition.  For f with |f'''| h^2 / 6 << f' the central
    difference at h = 1e-4 is off by ~1e-8 relative; the kernel's own error in fp32 is bounded by 1e-4 of sum |grad| |direction| here."""
    from diffphycon_amd import sequence as S
    g = _gen(11)
    n, m, D = 20, 30, 16
    q, k, v, w = (_randn(g, 1, r, 1, D) for r in (n, m, m, n))
    out, lse = S.attention_forward(q, k, v, causal=True)
    grads = S.attention_backward(w, q, k, v, out, lse, causal=True)

    def f(*x):
        return (O.attention(*(y[0, :, 0].double() for y in x), causal=True)["out"][0] * w[0, :, 0].double()).sum()
    O.UNIT[torch.float64], O.TINY[torch.float64] = 2.0 ** -53, 0.0
    x = [y.double() for y in (q, k, v)]
    for i in range(3):
        d = _randn(g, *x[i].shape).double()
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + 1e-4 * d, x[i] - 1e-4 * d
        want = (f(*up) - f(*down)) / 2e-4
        assert abs((grads[i].double() * d).sum() - want) <= 1e-4 * (grads[i].double().abs() * d.abs()).sum()


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16], ids=str)
def test_attention_small_gradients_and_large_scores(t, dev):
    """fp16 would lose gradients of 1e-6 and probabilities of 1e-5 without its scaling; large scores must not overflow."""
    from diffphycon_amd import sequence as S
    g = _gen(12)
    B, Lq, Lk, H, D = 1, 64, 900, 1, 64
    for qs, gs in ((0.01, 1e-4 if t == torch.float16 else 1e-20), (30.0, 1.0), (0.01, 300.0)):
        q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t, scale=qs), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t, scale=gs)
        out, lse = S.attention_forward(q, k, v)
        grads = S.attention_backward(dout, q, k, v, out, lse)
        _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)])


def test_attention_offsets_beyond_32_bits(dev):
    from diffphycon_amd import sequence as S
    g = _gen(13)
    L, H, D, t = 40, 1, 64, torch.bfloat16
    far = 2 ** 31 + 128
    big = torch.empty(far + L * H * D, dtype=t, device=dev)
    view = big.as_strided((2, L, H, D), (far, H * D, D, 1))
    k = _randn(g, 2, L, H, D, dtype=t)
    view.copy_(k)
    q, v, dout = (_randn(g, 2, L, H, D, dtype=t) for _ in range(3))
    out, lse = S.attention_forward(q, view, v)
    ref, _ = S.attention_forward(q, k, v)
    assert torch.equal(out, ref)
    for a, b in zip(S.attention_backward(dout, q, view, v, out, lse), S.attention_backward(dout, q, k, v, out, lse)):
        assert torch.equal(a, b)


def test_attention_empty_sizes(dev):
    from diffphycon_amd import sequence as S
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 5), (2, 5, 0), (2, 0, 0)):
        for causal in (False, True):
            q, k = torch.randn(B, Lq, 2, 32, device=dev), torch.randn(B, Lk, 2, 32, device=dev)
            out, lse = S.attention_forward(q, k, k, causal=causal)
            dq, dk, dv = S.attention_backward(q, q, k, k, out, lse, causal=causal)
            assert out.shape == q.shape and lse.shape == (B, 2, Lq) and dq.shape == q.shape and dk.shape == k.shape == dv.shape
            assert not out.any() and not dq.any() and not dk.any() and not dv.any()
            assert torch.isneginf(lse).all()


# ---------------------------------------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,C", [(1, 1), (3, 8), (5, 7), (64, 64), (700, 33), (64, 512), (17, 1000), (9, 1024), (6, 1027), (3, 2048), (5, 4096), (2, 8192), (3, 9000), (2, 20000), (3000, 16)])
def test_layer_norm(rows, C, t, dev):
    from diffphycon_amd import sequence as S
    g = _gen(rows * 31 + C)
    x, dy = _randn(g, rows, C, dtype=t, scale=2.0, shift=0.5), _randn(g, rows, C, dtype=t)
    for wt, with_b in ((t, True), (torch.float32, True), (None, False), (t, False)):
        w = _randn(g, C, dtype=wt, shift=1.0) if wt is not None else None
        b = _randn(g, C, dtype=wt) if with_b else None
        y, stats = S.layer_norm_forward(x, w, b, eps=1e-5)
        dx, dw, db = S.layer_norm_backward(dy, x, stats, w)
        r = O.layer_norm(x, w, b, 1e-5, dy, pt=wt or torch.float32)
        assert dw.dtype == (wt or torch.float32) == db.dtype
        for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db), ("mean", stats[:, :1]), ("rstd", stats[:, 1:])):
            _within(name, got, *r[name])


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("rows,C", [(2500, 1540), (1100, 2056), (1301, 4104), (1100, 4099), (1037, 8200), (700, 12008)])
def test_layer_norm_of_many_wide_rows(rows, C, t, dev):
    """More rows than workgroups, in every width of a group: the next row is on its way while one is worked on."""
    from diffphycon_amd import sequence as S
    g = _gen(rows)
    x, dy = _randn(g, rows, C, dtype=t, scale=1.5, shift=0.25), _randn(g, rows, C, dtype=t, scale=0.1)
    w, b = _randn(g, C, scale=0.1, shift=1.0).to(t), _randn(g, C).to(t)
    y, st = S.layer_norm_forward(x, w, b)
    dx, dw, db = S.layer_norm_backward(dy, x, st, w)
    r = O.layer_norm(x, w, b, 1e-5, dy, t)
    for name, got in (("y", y), ("mean", st[:, :1]), ("rstd", st[:, 1:]), ("dx", dx), ("dw", dw), ("db", db)):
        _within(name, got, *r[name])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_layer_norm_values(t, dev):
    """A mean far above the spread, constant rows, and rows of infinities or NaN next to ordinary ones."""
    from diffphycon_amd import sequence as S
    g = _gen(3)
    x = _randn(g, 12, 256, dtype=t, scale=0.25 if t == torch.float32 else 1.0, shift=100.0)
    x[3], x[4] = 5.0, 0.0
    dy = _randn(g, 12, 256, dtype=t)
    y, stats = S.layer_norm_forward(x)
    dx, dw, db = S.layer_norm_backward(dy, x, stats)
    r = O.layer_norm(x, None, None, 1e-5, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        _within(name, got, *r[name])
    bad = x.clone()
    bad[0, 3], bad[7, 0] = math.inf, math.nan
    yb, _ = S.layer_norm_forward(bad)
    keep = [i for i in range(12) if i not in (0, 7)]
    assert torch.equal(yb[keep], y[keep]) and yb[[0, 7]].isnan().all()


def test_layer_norm_layouts_and_empty(dev):
    from diffphycon_amd import sequence as S
    g = _gen(4)
    for t in TYPES:
        base = _randn(g, 6, 5, 96, dtype=t)
        for x in (base[:, :, 16:80], base.transpose(0, 1), base[:, ::2, 3:36], base.permute(2, 0, 1), base[:1, :1, :1].expand(4, 3, 32), base[:, 0, ::2]):
            dy = torch.randn(x.shape, generator=g).to(t).to(dev)
            y, st = S.layer_norm_forward(x)
            y2, st2 = S.layer_norm_forward(x.contiguous())
            assert torch.equal(y, y2) and torch.equal(st, st2) and y.shape == x.shape
            for a, b in zip(S.layer_norm_backward(dy.transpose(0, -2).contiguous().transpose(0, -2), x, st), S.layer_norm_backward(dy, x.contiguous(), st)):
                assert torch.equal(a, b)
            one = dy.flatten()[:x.shape[-1]].expand(x.shape)         # one gradient for all rows
            for a, b in zip(S.layer_norm_backward(one, x, st), S.layer_norm_backward(one.contiguous(), x.contiguous(), st)):
                assert torch.equal(a, b)
    x = torch.randn(0, 8, device=dev)
    y, st = S.layer_norm_forward(x)
    dx, dw, db = S.layer_norm_backward(x, x, st, torch.ones(8, device=dev))
    assert y.shape == x.shape == dx.shape and st.shape == (0, 2) and not dw.any() and not db.any()
    x = torch.randn(5, 8, device=dev)
    y, st = S.layer_norm_forward(x)
    assert S.layer_norm_backward(x, x, st, param_grads=False)[1:] == (None, None)


# ---------------------------------------------------------------------------------------------------------------- rotary
@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,T,H,Hk,D,R", [(1, 1, 1, 1, 2, 2), (2, 5, 3, 1, 32, 32), (3, 33, 4, 4, 64, 32), (1, 7, 5, 2, 10, 6), (2, 9, 2, 1, 128, 96), (1, 300, 2, 2, 80, 80), (2, 3, 1, 1, 128, 20)])
def test_rotary(B, T, H, Hk, D, R, layout, t, dev):
    from diffphycon_amd import sequence as S
    g = _gen(B * T + D)
    q, k = _randn(g, B, T, H, D, dtype=t), _randn(g, B, T, Hk, D, dtype=t)
    for scaling, factor in ((None, 1.0), ("linear", 4.0), ("ramp", 8.0)) + ((("ntk", 4.0),) if R > 2 else ()):
        table = S.RotaryTable(R, 70000, layout=layout, scaling=scaling, factor=factor, device=dev)
        pos = torch.randint(0, 70000, (B, T), generator=g).to(dev)
        for p, full in ((pos, pos), (pos[0].int(), pos[:1].expand(B, T)), (None, (torch.arange(T, device=dev) + 69000).expand(B, T))):
            kw = dict(positions=p) if p is not None else dict(start=69000)
            for f, transpose in ((S.rotary_forward, False), (S.rotary_backward, True)):
                yq, yk = f(q, k, table, **kw)
                for y, x in ((yq, q), (yk, k)):
                    _within("rotary", y, *O.rotary(x, full, table.frequencies, layout, table.attention_factor, transpose))
                assert torch.equal(f(q, None, table, **kw)[0], yq)
                a, b = q.clone(), k.clone()
                f(a, b, table, out=(a, b), **kw)
                assert torch.equal(a, yq) and torch.equal(b, yk)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("B,T,H,Hk,D,R", [(2, 4500, 13, 4, 80, 48), (1, 7, 3, 1, 512, 512), (1, 5, 2, 1, 1040, 1024), (3, 41, 5, 2, 264, 256), (1, 70, 9, 3, 24, 16), (1, 40, 4, 2, 27, 16)])
def test_rotary_of_many_tokens_and_of_long_and_odd_heads(B, T, H, Hk, D, R, layout, t, dev):
    from diffphycon_amd import sequence as S
    g = _gen(T + R)
    q, k = _randn(g, B, T, H, D, dtype=t), _randn(g, B, T, Hk, D, dtype=t)
    table = S.RotaryTable(R, T + 9, layout=layout, device=dev)
    full = (torch.arange(T, device=dev) + 9).expand(B, T)
    yq, yk = S.rotary_forward(q, k, table, start=9)
    for y, x in ((yq, q), (yk, k)):
        _within("rotary", y, *O.rotary(x, full, table.frequencies, layout))
    for in_q, in_k in ((True, True), (True, False), (False, True)):  # both in place, or one
        a, b = q.clone(), k.clone()
        oq, ok = a if in_q else torch.empty_like(a), b if in_k else torch.empty_like(b)
        S.rotary_forward(a, b, table, start=9, out=(oq, ok))
        assert torch.equal(oq, yq) and torch.equal(ok, yk)


def test_rotary_frequencies(dev):
    """The scalings against their definitions, by hand, at pairs where they differ."""
    from diffphycon_amd import sequence as S
    R, base = 64, 10000.0
    f = [base ** (-2 * i / R) for i in range(R // 2)]
    lin = S.RotaryTable(R, 16, scaling="linear", factor=4.0, device=dev).frequencies
    ntk = S.RotaryTable(R, 16, scaling="ntk", factor=4.0, device=dev).frequencies
    t = S.RotaryTable(R, 4096, scaling="ramp", factor=4.0, trained_positions=1024, device=dev)
    for i in (0, 7, 20, 31):
        assert math.isclose(lin[i], f[i] / 4, rel_tol=1e-14)
        assert math.isclose(ntk[i], (base * 4 ** (R / (R - 2))) ** (-2 * i / R), rel_tol=1e-13)
        c = min(1.0, max(0.0, (1024 * f[i] / (2 * math.pi) - 1) / 31))
        assert math.isclose(t.frequencies[i], (1 - c) * f[i] / 4 + c * f[i], rel_tol=1e-13)
    assert math.isclose(ntk[0], 1.0) and math.isclose(ntk[31], f[31] / 4, rel_tol=1e-12)          # fastest kept, slowest slowed by the factor
    assert math.isclose(t.attention_factor, 0.1 * math.log(4) + 1)


def test_rotary_layouts_and_bad_positions(dev):
    from diffphycon_amd import sequence as S
    g = _gen(21)
    for t in TYPES:
        for layout in ("interleaved", "half"):
            table = S.RotaryTable(16, 50, layout=layout, device=dev)
            qkv = _randn(g, 2, 6, 3, 4, 40, dtype=t)
            q, k, v = qkv.unbind(2)
            ref = S.rotary_forward(q.contiguous(), k.contiguous(), table, start=3)
            got = S.rotary_forward(q, k, table, start=3)
            assert all(torch.equal(a, b) for a, b in zip(ref, got))
            keep = v.clone()
            S.rotary_forward(q, k, table, start=3, out=(q, k))       # in place in the projection, the values untouched
            assert torch.equal(q, ref[0]) and torch.equal(k, ref[1]) and torch.equal(v, keep)
            flat = ref[0].flatten(0, 1)
            p = torch.tensor([0, 49, 50, -1, 2 ** 40, -2 ** 63, 1, 2, 3, 4, 5, 6], device=dev)
            y, _ = S.rotary_forward(flat, None, table, positions=p)
            bad = torch.tensor([False, False, True, True, True, True] + [False] * 6, device=dev)
            assert y[bad][..., :16].isnan().all() and torch.equal(y[bad][..., 16:], flat[bad][..., 16:])
            ok = _randn(g, 1, 12, 4, 40, dtype=t)[0]
            assert torch.equal(y[~bad], S.rotary_forward(flat[~bad], None, table, positions=p[~bad])[0]) and not y[~bad].isnan().any()
            with pytest.raises(ValueError):
                S.rotary_forward(q, k, table, out=(k, q))
            empty = S.rotary_forward(ok[:0], None, table)[0]
            assert empty.shape == (0, 4, 40)


# ---------------------------------------------------------------------------------------------------------------- together
def _block(S, x, w, wn, bn, table, H, Hk, D, dout, plan=None, mask=None):
    """A pre-norm attention block without output projection, forward and backward -> out and all gradients.  x [B, L, C]."""
    y, st = S.layer_norm_forward(x, wn, bn)
    B, L, _ = x.shape
    qkv = torch.matmul(y, w).view(B, L, H + 2 * Hk, D)
    q, k, v = qkv[:, :, :H], qkv[:, :, H:H + Hk], qkv[:, :, H + Hk:]
    q, k = S.rotary_forward(q, k, table)
    out, lse = S.attention_forward(q, k, v, causal=True, key_mask=mask)
    d = torch.empty_like(qkv)
    dq, dk, dv = d[:, :, :H], d[:, :, H:H + Hk], d[:, :, H + Hk:]
    S.attention_backward(dout, q, k, v, out, lse, causal=True, key_mask=mask, grads=(dq, dk, dv))
    S.rotary_backward(dq, dk, table, out=(dq, dk))
    d = d.view(B, L, -1)
    dw = torch.matmul(y.reshape(B * L, -1).t().contiguous(), d.reshape(B * L, -1))
    dx, dwn, dbn = S.layer_norm_backward(torch.matmul(d, w.t().contiguous()), x, st, wn)
    return out, dx, dw, dwn, dbn


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_block_against_autograd(layout, dev):
    """The operators in a run against torch's autograd of the same block in 64 bits.  fp32: the chain of sums of up to 192 (projection), 32 (scores) and 45
    (probabilities) terms is off by some 2^-24 * 300 ~ 2e-5 of the terms' sizes; 1e-4 of each gradient's largest entry is the bound."""
    from diffphycon_amd import sequence as S
    g = _gen(31)
    B, L, C, H, Hk, D = 2, 45, 192, 4, 2, 32
    x, w, wn, bn = _randn(g, B, L, C), _randn(g, C, (H + 2 * Hk) * D, scale=C ** -0.5), _randn(g, C, shift=1.0), _randn(g, C)
    dout = _randn(g, B, L, H, D)
    mask = torch.ones(B, L, dtype=torch.bool, device=dev)
    mask[1, 30:] = False
    table = S.RotaryTable(D, L, layout=layout, device=dev)
    got = _block(S, x, w, wn, bn, table, H, Hk, D, dout, mask=mask)
    leaves = [v.double().cpu().requires_grad_() for v in (x, w, wn, bn)]
    X, Wd, WN, BN = leaves
    qkv = (torch.nn.functional.layer_norm(X, (C,), WN, BN, 1e-5) @ Wd).view(B, L, H + 2 * Hk, D)
    ang = torch.arange(L, dtype=torch.float64)[:, None] * table.frequencies
    co, si = ang.cos()[None, :, None], ang.sin()[None, :, None]
    a, b = (qkv[..., 0::2], qkv[..., 1::2]) if layout == "interleaved" else (qkv[..., :D // 2], qkv[..., D // 2:])
    pair = (a * co - b * si, a * si + b * co)
    turned = torch.stack(pair, -1).flatten(-2) if layout == "interleaved" else torch.cat(pair, -1)
    q, k, v = turned[:, :, :H], turned[:, :, H:H + Hk].repeat_interleave(H // Hk, 2), qkv[:, :, H + Hk:].repeat_interleave(H // Hk, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    s = s.masked_fill(~(torch.ones(L, L, dtype=torch.bool).tril() & mask.cpu()[:, None, None, :]), -math.inf)
    out = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v)
    grads = torch.autograd.grad((out * dout.double().cpu()).sum(), leaves)
    for name, y, r in zip(("out", "dx", "dw", "dwn", "dbn"), got, (out,) + grads):
        r = r.detach()
        assert (y.cpu().double() - r).abs().max() <= 1e-4 * r.abs().max(), name


def test_block_in_a_graph_on_another_stream_and_twice(dev):
    """Captured and replayed with new inputs, beside eager work and a second graph: equal to eager calls bit for bit, every replay."""
    from diffphycon_amd import sequence as S
    g = _gen(32)
    B, L, C, H, Hk, D = 2, 130, 128, 4, 2, 64
    t = torch.bfloat16
    w, wn, bn = _randn(g, C, (H + 2 * Hk) * D, dtype=t, scale=C ** -0.5), _randn(g, C, dtype=t, shift=1.0), _randn(g, C, dtype=t)
    table = S.RotaryTable(D, L, layout="half", device=dev)
    plan = S.SequencePlan.packed([1, 100, 159], device=dev)

    def work(x, dout):
        y, st = S.layer_norm_forward(x, wn, bn)
        q, k = S.rotary_forward(y.view(B, L, 2, D), y.view(B, L, 2, D), table)
        out, lse = S.attention_forward(q, k, q, causal=True)
        o2, l2 = S.attention_forward(q.flatten(0, 1), k.flatten(0, 1), q.flatten(0, 1), causal=True, plan=plan)
        gr = S.attention_backward(dout, q, k, q, out, lse, causal=True) + S.attention_backward(dout.flatten(0, 1), q.flatten(0, 1), k.flatten(0, 1), q.flatten(0, 1), o2, l2, causal=True, plan=plan)
        return (y, out, lse, o2, *gr, *S.layer_norm_backward(y, x, st, wn))

    static = [(_randn(g, B, L, C, dtype=t), _randn(g, B, L, 2, D, dtype=t)) for _ in range(2)]
    work(*static[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = work(*s)
        graphs.append(gr)
        outs.append(o)
    for it in range(3):
        for s in static:
            for x in s:
                x.copy_(_randn(g, *x.shape, dtype=t))
        want = [[y.clone() for y in work(*s)] for s in static]
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, r)), it
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = work(*static[0])
    here = work(*static[1])                                          # (two calls at once on two streams)
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want[0])) and all(torch.equal(a, b) for a, b in zip(here, want[1]))


def test_drawn_sizes(dev):
    """Sizes nobody chose: lengths, heads, head sizes, masks at random (seeded)."""
    from diffphycon_amd import sequence as S
    rng = random.Random(2)
    for case in range(30):
        g = _gen(case)
        t = rng.choice(TYPES)
        Hk, G, D = rng.randint(1, 3), rng.choice((1, 2, 3)), 8 * rng.randint(1, 16)
        Lq, Lk, B, causal = rng.randint(1, 300), rng.randint(1, 300), rng.randint(1, 3), rng.random() < 0.5
        q, k, v, dout = _randn(g, B, Lq, Hk * G, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, Hk * G, D, dtype=t)
        mask = (torch.rand(B, Lk, generator=g) < 0.7).to(dev) if rng.random() < 0.4 else None
        print(case, t, B, Lq, Lk, Hk, G, D, causal, mask is not None, flush=True)
        out, lse = S.attention_forward(q, k, v, causal=causal, key_mask=mask)
        grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, key_mask=mask)
        _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)] * B, causal=causal, mask=mask)


def test_single_tokens_in_a_graph(dev):
    """A step's attention over masked keys, captured with its splits and joins: every replay equals the eager call on what the cache then holds."""
    from diffphycon_amd import sequence as S
    g = _gen(51)
    B, Lk, H, Hk, D = 3, 2500, 8, 2, 128
    q, k, v = (_randn(g, B, n, h, D, dtype=torch.bfloat16) for n, h in ((1, H), (Lk, Hk), (Lk, Hk)))
    mask = torch.zeros(B, Lk, dtype=torch.bool, device=dev)
    S.attention_forward(q, k, v, key_mask=mask)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, lse = S.attention_forward(q, k, v, key_mask=mask)
    for n in (0, 1, 33, 1024, 2500):
        mask[:, :n] = True
        if n == 1024:
            mask[1, 5:900] = False
        q.copy_(_randn(g, *q.shape, dtype=q.dtype))
        want = S.attention_forward(q, k, v, key_mask=mask)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and lse.isinf().all() == (n == 0)
        for b in range(B):
            for h in range(H):
                r = O.attention(q[b, :, h], k[b, :, h // 4], v[b, :, h // 4], mask=mask[b])
                _within("out", out[b, :, h], *r["out"])
                _within("lse", lse[b, h], *r["lse"])


def test_tables_are_refused_in_a_capture(dev):
    from diffphycon_amd import sequence as S
    x = torch.ones(4, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="before the capture"):
            S.RotaryTable(8, 16)
        with pytest.raises(RuntimeError, match="before the capture"):
            S.SequencePlan.packed([3, 4])
        y = x + 1
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, x + 1)
