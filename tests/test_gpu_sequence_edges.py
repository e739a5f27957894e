"""diffphycon_amd.sequence where a call is allowed but unusual, against the definitions in 64 bits (tests/sequence_oracle.py)."""
import math

import pytest
import torch

import sequence_oracle as O
from test_gpu_sequence import TYPES, _check_attention, _gen, _randn, _within, dev  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("C", [8, 32, 128, 512, 2048, 16384, 32768])
@pytest.mark.parametrize("pad", [0, 1])
def test_layer_norm_gradient_of_a_far_constant_row(C, pad, t, dev):
    """Rows of 2^100: x - mean is 0, while mean / sqrt(eps) is beyond fp32's range; lanes past the row's end must not bring that in.  With xh = 0 the
    gradient is rstd (g - mean(g)), off by a sum of C terms and a few operations."""
    from diffphycon_amd import sequence as S
    g = _gen(C)
    x = torch.full((5, C + pad), 2.0 ** 100, dtype=t, device=dev)[:, :C]
    dy, w = _randn(g, 5, C, dtype=t), _randn(g, C, dtype=t, shift=1.0)
    y, st = S.layer_norm_forward(x, w, eps=1e-20)
    assert not y.any()
    dx, dw, db = S.layer_norm_backward(dy, x, st, w)
    z = dy.double() * w.double()
    rstd, mean, size = 1e-20 ** -0.5, z.mean(1, keepdim=True), z.abs().mean(1, keepdim=True)
    value = rstd * (z - mean)
    _within("dx", dx, value, O.add_rounding(value, rstd * O.E * (6 * z.abs() + (C + 10) * size), t))
    assert not dw.any()
    _within("db", db, dy.double().sum(0), O.add_rounding(dy.double().sum(0), 9 * O.E * dy.double().abs().sum(0), t))


# ---------------------------------------------------------------------------------------------------------------- attention: few keys under a mask
def _few(B, Lk, seen, seed):
    """A mask that leaves `seen` keys of Lk in each batch entry, spread over all of them."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros(B, Lk, dtype=torch.bool)
    for b in range(B):
        mask[b, torch.randperm(Lk, generator=g)[:seen]] = True
    return mask


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("seen", [1, 2, 5, 20, 60])
def test_attention_gradients_of_few_keys_under_a_mask(seen, D, t, dev):
    """Few keys among many: the gradients are as exact as those of a short sequence.  Once with the keys split over workgroups, once with the card full."""
    from diffphycon_amd import sequence as S
    for B, H, Hk in ((3, 4, 2), (40, 10, 10)):
        Lq, Lk = 30, 900
        g = _gen(seen + D)
        mask = _few(B, Lk, seen, seen).to(dev)
        q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
        k[~mask], v[~mask] = math.nan, math.inf
        out, lse = S.attention_forward(q, k, v, key_mask=mask)
        dq, dk, dv = S.attention_backward(dout, q, k, v, out, lse, key_mask=mask)
        for b in sorted({0, 1, B - 1}):
            for hk in range(Hk):
                sums = None
                for h in range(hk * (H // Hk), (hk + 1) * (H // Hk)):
                    r = O.attention(q[b, :, h], k[b, :, hk], v[b, :, hk], dout[b, :, h], mask=mask[b], swept=True, parts=True)
                    _within("dq", dq[b, :, h], r["dq"][0], O.add_rounding(*r["dq"], t))
                    part = [*r["dk"], *r["dv"]]
                    sums = part if sums is None else [x + y for x, y in zip(sums, part)]
                chain = (H // Hk) * O.E * Lq
                _within("dk", dk[b, :, hk], sums[0], O.add_rounding(sums[0], sums[1] * (1 + chain), t))
                _within("dv", dv[b, :, hk], sums[2], O.add_rounding(sums[2], sums[3] * (1 + chain), t))


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
@pytest.mark.parametrize("D,H,Hk", [(32, 2, 2), (64, 6, 2), (128, 2, 1)])
def test_attention_gradients_behind_left_padding(D, H, Hk, t, dev):
    """Causal sequences that start behind padding: their first rows see one key, two keys, ...  A block sees at most the real tokens."""
    from diffphycon_amd import sequence as S
    L, first = 700, [690, 640, 500, 447, 130]
    B = len(first)
    g = _gen(D)
    q, k, v, dout = _randn(g, B, L, H, D, dtype=t), _randn(g, B, L, Hk, D, dtype=t), _randn(g, B, L, Hk, D, dtype=t), _randn(g, B, L, H, D, dtype=t)
    mask = (torch.arange(L)[None] >= torch.tensor(first)[:, None]).to(dev)
    k[~mask], v[~mask] = math.nan, math.inf
    out, lse = S.attention_forward(q, k, v, causal=True, key_mask=mask)
    dq, dk, dv = S.attention_backward(dout, q, k, v, out, lse, causal=True, key_mask=mask)
    for b, f in enumerate(first):
        last = L if L - f <= 256 else 256                            # rows of blocks that see at most 256 keys
        for h in range(H):
            r = O.attention(q[b, :, h], k[b, :, h // (H // Hk)], v[b, :, h // (H // Hk)], dout[b, :, h], True, mask=mask[b], swept=True, parts=L - f <= 64)
            _within("dq", dq[b, :last, h], *(x[:last] for x in (r["dq"][0], O.add_rounding(*r["dq"], t))))
        assert not dq[b, :f].any() and not dk[b, :f].any() and not dv[b, :f].any()
    _check_attention(q.masked_fill(~mask[:, :, None, None], 0.0), k, v, dout.masked_fill(~mask[:, :, None, None], 0.0), out, lse, (dq, dk, dv), [(L, L)] * B, causal=True, mask=mask)


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
def test_attention_gradients_of_few_keys_are_the_same_masked_and_packed(t, dev):
    """The keys that a mask leaves, gathered into a plan's sequences: either way the gradients are rounded once, from values some 2 u^2 of their terms
    apart (u: half a step).  Such a pair rounds apart in a share u k of the elements (k: terms over result, below 16), by 2 u: 2 u (u k)^(1/2) < u / 2 in norm."""
    from diffphycon_amd import sequence as S
    B, Lq, Lk, H, D, seen = 4, 25, 1300, 3, 64, 7
    g = _gen(77)
    mask = _few(B, Lk, seen, 3).to(dev)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    out, lse = S.attention_forward(q, k, v, key_mask=mask)
    a = S.attention_backward(dout, q, k, v, out, lse, key_mask=mask)
    plan = S.SequencePlan.packed([Lq] * B, [seen] * B, device=dev)
    p = [q.flatten(0, 1), k[mask], v[mask]]
    out, lse = S.attention_forward(*p, plan=plan)
    b = S.attention_backward(dout.flatten(0, 1), *p, out, lse, plan=plan)
    for x, y in ((a[0].flatten(0, 1), b[0]), (a[1][mask], b[1]), (a[2][mask], b[2])):
        x, y = x.double(), y.double()
        assert ((x - y).norm() / y.norm()).item() <= O.UNIT[t] / 2


@pytest.mark.parametrize("t", TYPES[1:], ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_attention_key_gradients_of_few_queries_behind_left_padding(D, t, dev):
    """A key behind left padding is seen by as many queries as there are real tokens from it on: sums of few terms, however long the axis is."""
    from diffphycon_amd import sequence as S
    L, first, H, Hk = 500, [498, 490, 470], 4, 2
    B = len(first)
    g = _gen(D)
    q, k, v, dout = _randn(g, B, L, H, D, dtype=t), _randn(g, B, L, Hk, D, dtype=t), _randn(g, B, L, Hk, D, dtype=t), _randn(g, B, L, H, D, dtype=t)
    mask = (torch.arange(L)[None] >= torch.tensor(first)[:, None]).to(dev)
    out, lse = S.attention_forward(q, k, v, causal=True, key_mask=mask)
    dq, dk, dv = S.attention_backward(dout, q, k, v, out, lse, causal=True, key_mask=mask)
    for b in range(B):
        for hk in range(Hk):
            sums = None
            for h in (2 * hk, 2 * hk + 1):
                r = O.attention(q[b, :, h], k[b, :, hk], v[b, :, hk], dout[b, :, h], True, mask=mask[b], swept=True, parts=True)
                part = [*r["dk"], *r["dv"]]
                sums = part if sums is None else [x + y for x, y in zip(sums, part)]
            chain = 2 * O.E * L
            _within("dk", dk[b, :, hk], sums[0], O.add_rounding(sums[0], sums[1] * (1 + chain), t))
            _within("dv", dv[b, :, hk], sums[2], O.add_rounding(sums[2], sums[3] * (1 + chain), t))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_attention_gradients_of_an_infinite_row_do_not_depend_on_a_mask(bad, t, dev):
    """A row whose log-sum-exp is +inf (scores that overflowed, as torch.logsumexp gives it) or NaN takes part: with a mask that lets every key through dk and
    dv are what they are without one.  Only -inf is a row that sees nothing."""
    from diffphycon_amd import sequence as S
    g = _gen(81)
    B, Lq, Lk, H, D = 2, 40, 300, 2, 64
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lk, H, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    out, lse = S.attention_forward(q, k, v)
    q[0, 7, 1], lse[0, 1, 7] = math.inf, bad
    plain = S.attention_backward(dout, q, k, v, out, lse)
    masked = S.attention_backward(dout, q, k, v, out, lse, key_mask=torch.ones(B, Lk, dtype=torch.bool, device=dev))
    for x, y in zip(plain, masked):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
    assert plain[1][0, :, 1].isnan().all() and not plain[1][1].isnan().any()
    lse[0, 1, 7] = -math.inf
    masked = S.attention_backward(dout, q, k, v, out, lse, key_mask=torch.ones(B, Lk, dtype=torch.bool, device=dev))
    assert not any(x.isnan().any() for x in masked) and not masked[0][0, 7, 1].any()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("H,Hk,D", [(6, 2, 64), (2, 2, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_few_sequences_in_a_long_buffer(H, Hk, D, causal, t, dev):
    """Long and short sequences of a padded plan whose walks are split: partial sums are numbered by the blocks that the plan has."""
    from diffphycon_amd import sequence as S
    ql, kl, Lq, Lk = [1100, 3, 0, 140, 1], [1500, 700, 9, 140, 0], 1300, 1600
    B = len(ql)
    g = _gen(H + D)
    q, k, v, dout = _randn(g, B, Lq, H, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lk, Hk, D, dtype=t), _randn(g, B, Lq, H, D, dtype=t)
    plan = S.SequencePlan.padded(ql, Lq, kl, Lk, device=dev)
    out, lse = S.attention_forward(q, k, v, causal=causal, plan=plan)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, plan=plan)
    _check_attention(q, k, v, dout, out, lse, grads, list(zip(ql, kl)), causal=causal)
    plan = S.SequencePlan.padded([1] * B, Lq, kl, Lk, device=dev)    # one token a sequence: few rows, many splits
    out, lse = S.attention_forward(q, k, v, causal=causal, plan=plan)
    _check_attention(q, k, v, None, out, lse, None, list(zip([1] * B, kl)), causal=causal)


@pytest.mark.parametrize("far", [2 ** 25 - 128, 2 ** 25 - 64, 2 ** 25 - 48, 2 ** 25 - 16, 2 ** 25])
def test_attention_of_tokens_far_apart(far, dev):
    """Token strides at the border of what a kernel reads in place (bytes): the same results, to the bit, as from contiguous tensors."""
    from diffphycon_amd import sequence as S
    g = _gen(91)
    t, L, D = torch.bfloat16, 70, 64
    k, q, dout = (_randn(g, 1, L, 1, D, dtype=t) for _ in range(3))
    wide = torch.empty(L * far // 2, dtype=t, device=dev).as_strided((1, L, 1, D), (0, far // 2, D, 1))
    wide.copy_(k)
    out, lse = S.attention_forward(q, k, k, causal=True)
    o2, l2 = S.attention_forward(q, wide, wide, causal=True)
    assert torch.equal(out, o2) and torch.equal(lse, l2)
    for a, b in zip(S.attention_backward(dout, q, k, k, out, lse, causal=True), S.attention_backward(dout, q, wide, wide, out, lse, causal=True)):
        assert torch.equal(a, b)


def test_layer_norm_of_a_very_wide_row(dev):
    """2^27 + 264 columns: the parameters' gradients have more columns than one launch has threads for a column each."""
    from diffphycon_amd import sequence as S
    n = 2 ** 27 + 264
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(1, n, generator=g, device=dev).to(torch.bfloat16)
    dy = torch.randn(1, n, generator=g, device=dev).to(torch.bfloat16)
    y, st = S.layer_norm_forward(x)
    dx, dw, db = S.layer_norm_backward(dy, x, st)
    assert torch.equal(db, dy[0].float())                            # (one row: its own elements)
    xh = (x[0].float() - st[0, 0]) * st[0, 1]
    assert ((dw - dy[0].float() * xh).abs() <= 4 * O.E * dw.abs() + 1e-37).all()
    assert ((y[0].float() - xh).abs() <= O.UNIT[torch.bfloat16] * xh.abs() * 1.001 + 1e-37).all()
    assert abs(st[0, 0].item() - x.double().mean().item()) < 1e-6
    # dx: a lane adds at most n / 256 + 8 terms one by one, so a mean over the row is off by less than that many 2^-24 of its terms' mean size.  (That the
    # elements of dx add up to 0 is lost in their rounding: g lies on bf16's grid, and mean(g), 2^-13 here, is less than its step.)
    gx = dy[0].double() * xh.double()
    a, b, rstd = dy.double().mean(), gx.mean(), st[0, 1].double()
    off = (n / 256 + 24) * O.E * rstd * (dy.double().abs().mean() + xh.double().abs() * gx.abs().mean())
    value = rstd * (dy[0].double() - a - xh.double() * b)
    assert ((dx[0].double() - value).abs() <= O.UNIT[torch.bfloat16] * (value.abs() + off) + off + 8 * O.E * (dy[0].double().abs() + 1)).all()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("Lq,Lk", [(1, 8), (1, 2000), (60, 64), (200, 1500)])
@pytest.mark.parametrize("score", [127, 101, 60, 41, 33, 8])
def test_attention_scores_beyond_fp32_are_not_rows_that_see_nothing(score, Lq, Lk, t, dev):
    """A row of equal scores 1.75 * 2^score.  The first overflows when it is counted in powers of two, the others are further from a whole step of fp32 than
    an exponent reaches: NaN, in the row alone, never the zeros and -inf of a row without keys.  The last is ordinary: the keys share the row."""
    from diffphycon_amd import sequence as S
    g = _gen(95)
    q, k, v = (_randn(g, 1, n, 2, 16, dtype=t) for n in (Lq, Lk, Lk))
    row = Lq // 2
    k[0, :, 1, 0] = 1.75 * 2.0 ** (score // 2)
    q[0, :, 1, 0], q[0, row, 1] = 0.0, 0.0
    q[0, row, 1, 0] = 2.0 ** (score - score // 2)
    out, lse = S.attention_forward(q, k, v, scale=1.0)
    mean = v[0, :, 1].double().mean(0)
    if score == 8:
        assert ((out[0, row, 1].double() - mean).abs() <= 0.02).all() and abs(lse[0, 1, row].item() - 448 - math.log(Lk)) <= 1e-3
    else:
        assert not torch.isneginf(lse[0, 1, row]) and (lse[0, 1, row].isnan() or score < 127)
        assert out[0, row, 1].isnan().all() or ((out[0, row, 1].double() - mean).abs() <= 0.02).all()
    out[0, row, 1], lse[0, 1, row] = 0.0, 0.0
    assert out.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("B,H,Hk,Lq,Lk,D,causal", [
    (4, 2, 2, 641, 641, 64, True), (8, 4, 2, 769, 769, 32, True), (2, 4, 4, 1100, 1100, 128, True), (1, 16, 8, 641, 1100, 96, True),          # split walks
    (16, 8, 8, 641, 641, 32, True), (32, 8, 8, 513, 200, 32, True), (8, 8, 8, 1100, 1100, 64, True), (2, 16, 8, 1300, 257, 64, True),         # whole ones
    (8, 2, 2, 700, 1030, 64, False), (16, 16, 8, 300, 513, 32, False),
])
def test_attention_blocks_of_many_pairs(B, H, Hk, Lq, Lk, D, causal, t, dev):
    """(sequence, key head) pairs by the eight, whose blocks follow each other on one XCD, under a causal mask in bands (5 to 11 blocks: bands of 2 and 3, the
    last one shorter): every block is computed, with and without splits of the walks.  Buffers hold NaN before."""
    from diffphycon_amd import sequence as S
    g = _gen(Lq + D + B)
    q, k, v, dout = (torch.randn(B, n, h, D, generator=g).to(t).to(dev) for n, h in ((Lq, H), (Lk, Hk), (Lk, Hk), (Lq, H)))
    out = torch.full_like(q, math.nan)
    _, lse = S.attention_forward(q, k, v, causal=causal, out=out)
    grads = tuple(torch.full_like(x, math.nan) for x in (q, k, v))
    S.attention_backward(dout, q, k, v, out, lse, causal=causal, grads=grads)
    _check_attention(q, k, v, dout, out, lse, grads, [(Lq, Lk)] * B, causal=causal)


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "save"])
def test_copies_of_tables_and_plans_stand_alone(how, dev, tmp_path):
    """A copied model copies its RotaryTable and SequencePlan: the copies read their own memory, when the originals are gone too, on any stream."""
    import copy
    import pickle

    from diffphycon_amd import sequence as S

    def copied(x):
        if how == "deepcopy":
            return copy.deepcopy(x)
        if how == "pickle":
            return pickle.loads(pickle.dumps(x))
        torch.save(x, tmp_path / "x.pt")
        return torch.load(tmp_path / "x.pt", weights_only=False)     # (a file this test wrote)

    g = _gen(99)
    q, k, v, dout = (_randn(g, 200, 2, 64, dtype=torch.bfloat16) for _ in range(4))
    table, plan = S.RotaryTable(64, 300, layout="half", device=dev), S.SequencePlan.packed([150, 0, 50], device=dev)
    turned = S.rotary_forward(q, k, table, start=7)
    out, lse = S.attention_forward(*turned, v, causal=True, plan=plan)
    grads = S.attention_backward(dout, *turned, v, out, lse, causal=True, plan=plan)
    t2, p2 = copied(table), copied(plan)
    assert t2.table.data_ptr() != table.table.data_ptr() and p2.table.data_ptr() != plan.table.data_ptr()
    table.table.fill_(math.nan)                                      # (the originals' memory means something else by now)
    plan.table.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            again = S.rotary_forward(q, k, t2, start=7)
            o2, l2 = S.attention_forward(*again, v, causal=True, plan=p2)
            g2 = S.attention_backward(dout, *again, v, o2, l2, causal=True, plan=p2)
        torch.cuda.synchronize()
        for a, b in zip((*turned, out, lse, *grads), (*again, o2, l2, *g2)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("H,Hk,D", [(4, 2, 64), (3, 3, 128), (2, 1, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_of_keys_far_apart(H, Hk, D, causal, t, dev):
    """1 to 256 keys among 4500, which are gathered (257 are not), in packed sequences that start anywhere: the masks' bytes lie on no boundary.  Under the causal
    mask rows of one block see different numbers of them."""
    from diffphycon_amd import sequence as S
    ql, kl, seen = [300, 37, 200, 130, 64, 1], [4500, 4097, 1301, 700, 263, 300], [256, 3, 130, 65, 64, 257]
    g = _gen(D + H)
    q, k, v, dout = _randn(g, sum(ql), H, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(kl), Hk, D, dtype=t), _randn(g, sum(ql), H, D, dtype=t)
    mask = torch.cat([_few(1, nk, n, nk)[0] for nk, n in zip(kl, seen)]).to(dev)
    k[~mask], v[~mask] = math.nan, math.inf
    plan = S.SequencePlan.packed(ql, kl, device=dev)
    out, lse = S.attention_forward(q, k, v, causal=causal, key_mask=mask, plan=plan)
    grads = S.attention_backward(dout, q, k, v, out, lse, causal=causal, key_mask=mask, plan=plan)
    _check_attention(q, k, v, dout, out, lse, grads, list(zip(ql, kl)), packed=True, causal=causal, mask=mask)
    few = 64 if t == torch.float32 else 256
    q0 = k0 = 0
    for nq, nk, n in zip(ql, kl, seen):
        for h in range(H):
            a, b = (slice(q0, q0 + nq), h), (slice(k0, k0 + nk), h // (H // Hk))
            if n <= few:
                r = O.attention(q[a], k[b], v[b], dout[a], causal, mask=mask[k0:k0 + nk], swept=True, parts=n <= 64)
                _within("dq", grads[0][a], r["dq"][0], O.add_rounding(*r["dq"], t))
        q0, k0 = q0 + nq, k0 + nk
